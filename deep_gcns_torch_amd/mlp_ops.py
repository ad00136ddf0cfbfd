"""The node-wise MLP in 32, 16 and 8 bits: root-mean-square norm with the residual's addition, and the product with bias,
activation and residual in its epilogue (csrc/rms_norm.hip, csrc/linear_act.hip).

``node_ops`` holds the fp32 row operators that the reference's own models use; these are the ones around them for models
whose rows are wider than 256 channels, or kept in bf16, fp16 or 8 bits:

    h = x + r;  y = h * rsqrt(mean(h^2) + eps) * w     rms_norm_rows(x, w, eps, residual=r)        forward and backward
    the same y as e4m3 rows, one fp32 scale each       rms_norm_rows_e4m3(x, w, eps, residual=r)   forward
    x as e4m3 rows                                     quantize_rows(x)                            forward
    act(x W^T + b) + r                                 linear_act(x, W, b, act, residual=r)        forward and backward
    the same of e4m3 rows and an e4m3 weight           linear_act_e4m3(x, W, b, act, residual=r)   forward

Rows are the last dimension; leading dimensions are free and may be empty.  Sums and statistics are fp32, every result is
rounded once to its type.  Work runs on the current stream of the inputs' device; results do not depend on timing (no
atomics).  What an operator does not take raises, nothing falls back.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["ACTIVATIONS", "RMSNorm", "RowsE4M3", "linear_act", "linear_act_e4m3", "quantize_rows", "rms_norm_rows",
           "rms_norm_rows_e4m3"]

#: activation name -> code (include/dgcn.h)
ACTIVATIONS = {"none": 0, "relu": 1, "leakyrelu": 2, "gelu": 3, "silu": 4}
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_E4M3 = 3
_MAX_NORM_C = 32768
_MAX_K = 1 << 20


class RowsE4M3(NamedTuple):
    """Rows in 8 bits: the row's values are ``data * scale``.  ``data`` (..., C) ``torch.float8_e4m3fn``, ``scale`` (...)
    fp32."""
    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        return (self.data.to(torch.float32) * self.scale.unsqueeze(-1)).to(dtype)


# The calls below are made once per layer and token: checks and launches are written to touch each argument once.
def _device(what: str, *tensors) -> int:
    """Index of the device that all of the tensors (None apart) are on."""
    d = tensors[0].get_device()
    for t in tensors:
        if t is not None and (d < 0 or t.get_device() != d):
            _lib.require_device(*tensors)        # raises: a CPU tensor, or two devices
    return d


def _row_type(x: torch.Tensor, what: str) -> int:
    t = _TYPES.get(x.dtype)
    if t is None:
        raise TypeError(f"{what}: rows must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError(f"{what}: rows need a last dimension of at least 1, got {tuple(x.shape)}")
    return t


def _rows2d(x: torch.Tensor):
    """``x`` as (rows, C) with unit stride in a row, and its row stride.  Rows that repeat (stride 0) are taken as they are."""
    C = x.size(-1)
    x2 = x if x.dim() == 2 else x.reshape(-1, C)
    ld, inner = x2.stride()
    if (inner != 1 and C > 1) or ld < 0:
        x2 = x2.contiguous()
        ld = C
    return x2, ld if x2.size(0) > 1 else C


def _param(p, n: int, dtype, what: str):
    """A (n,) parameter in the rows' type or fp32 -> (contiguous tensor, is it fp32)."""
    if p is None:
        return None, 0
    if p.dim() != 1 or p.size(0) != n:
        raise ValueError(f"{what} must have shape ({n},), got {tuple(p.shape)}")
    if p.dtype != dtype and p.dtype != torch.float32:
        raise TypeError(f"{what} must be {dtype} or float32, got {p.dtype}")
    return p if p.is_contiguous() else p.detach().contiguous(), 1 if p.dtype == torch.float32 else 0


def _same_rows(r, x: torch.Tensor, n: int, dtype, what: str) -> None:
    want = (*x.shape[:-1], n)
    if r.shape != want:
        raise ValueError(f"{what} must have shape {tuple(want)}, got {tuple(r.shape)}")
    if r.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, got {r.dtype}")


def _needs_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_grad_only(what, *tensors):
    if _needs_grad(*tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or on tensors that require none")


# ---- root-mean-square norm ------------------------------------------------------------------------------------------
def _rms(what, x, weight, eps, residual, e4m3: bool, want_rstd: bool):
    """Checks and launch -> (y or RowsE4M3, h or None, rstd or None), contiguous, of x's shape."""
    t = _row_type(x, what)
    C = x.size(-1)
    if C > _MAX_NORM_C:
        raise ValueError(f"{what}: rows of at most {_MAX_NORM_C} channels, got {C}")
    w, w_f32 = _param(weight, C, x.dtype, "weight")
    shape = x.shape
    if residual is not None:
        if residual.shape != shape or residual.dtype != x.dtype:
            _same_rows(residual, x, C, x.dtype, "residual")
    d = _device(what, x, weight, residual)
    x2, ldx = _rows2d(x)
    rows = x2.size(0)
    h = rstd = y = q = scale = None
    r2, ldr = (None, 0) if residual is None else _rows2d(residual)
    if residual is not None:
        h = x.new_empty(shape)
    if want_rstd:
        rstd = x.new_empty(rows, dtype=torch.float32)
    if e4m3:
        q = x.new_empty(shape, dtype=torch.float8_e4m3fn)
        scale = x.new_empty(shape[:-1], dtype=torch.float32)
    else:
        y = x.new_empty(shape)
    if rows:
        ptr = _lib.ptr
        with _lib.device_ctx(d):
            rc = _lib.load().dgcn_rms_norm_fwd(x2.data_ptr(), ldx, ptr(r2), ldr, ptr(w), w_f32, eps, t, ptr(y), ptr(h), ptr(q),
                                               ptr(scale), ptr(rstd), rows, C, _lib.current_stream_handle(d))
        if rc:
            _lib.check(rc, "dgcn_rms_norm_fwd")
    return (RowsE4M3(q, scale) if e4m3 else y), h, rstd


class _RMSNormRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps: float):
        ctx.set_materialize_grads(False)
        y, h, rstd = _rms("rms_norm_rows", x, weight, eps, residual, False, True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, g, gh=None):
        h, weight, rstd = ctx.saved_tensors
        need_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[2]
        need_w = weight is not None and ctx.needs_input_grad[1]
        if g is None or h.numel() == 0:          # only the sum was used: its gradient is both inputs'
            gh = torch.zeros_like(h) if gh is None else gh
            gw = torch.zeros_like(weight) if need_w else None
            return (gh if ctx.needs_input_grad[0] else None), gw, (gh if ctx.needs_input_grad[2] else None), None
        lib = _lib.load()
        d = h.get_device()
        h2, ldh = _rows2d(h)
        g2, ldg = _rows2d(g)
        gh2, ldgh = (None, 0) if gh is None else _rows2d(gh)
        rows, C = h2.shape
        w, w_f32 = _param(weight, C, h.dtype, "weight")
        dx = h.new_empty(h.shape) if need_x else None
        gw = parts = None
        if need_w:
            gw = weight.new_empty(C)
            parts = h.new_empty((lib.dgcn_rms_norm_num_partials(rows, C), C), dtype=torch.float32)
        if need_x or need_w:
            ptr = _lib.ptr
            with _lib.device_ctx(d):
                rc = lib.dgcn_rms_norm_bwd(g2.data_ptr(), ldg, ptr(gh2), ldgh, h2.data_ptr(), ldh, ptr(w), w_f32,
                                           rstd.data_ptr(), _TYPES[h.dtype], ptr(dx), ptr(gw), ptr(parts), rows, C,
                                           _lib.current_stream_handle(d))
            if rc:
                _lib.check(rc, "dgcn_rms_norm_bwd")
        return (dx if ctx.needs_input_grad[0] else None), gw, (dx if ctx.needs_input_grad[2] else None), None


def rms_norm_rows(x, weight=None, eps: float = 1e-6, residual=None):
    """``h = x [+ residual]``, ``y = h * rsqrt(mean(h^2) + eps) [* weight]`` over the last dimension.

    Returns ``y``, or ``(y, h)`` with a residual: ``h`` is the stream that the next layer adds to.  ``x`` (..., C) fp32,
    bf16 or fp16, C <= 32768; ``residual`` of the same shape and type; ``weight`` (C,) in the rows' type or fp32.  ``y`` is
    computed from the fp32 sum; its gradient (of x, weight and residual) from the stored ``h``."""
    if _needs_grad(x, weight, residual):
        return _RMSNormRows.apply(x, weight, residual, eps)
    y, h, _ = _rms("rms_norm_rows", x, weight, eps, residual, False, False)
    return y if residual is None else (y, h)


def rms_norm_rows_e4m3(x, weight=None, eps: float = 1e-6, residual=None):
    """``rms_norm_rows`` whose ``y`` leaves as :class:`RowsE4M3`: ``scale = max|y| / 448`` per row (1 for a row of zeros).
    Returns the rows, or ``(rows, h)`` with a residual.  A NaN or an infinity becomes NaN in its own place.  No gradient."""
    _no_grad_only("rms_norm_rows_e4m3", x, weight, residual)
    y, h, _ = _rms("rms_norm_rows_e4m3", x, weight, eps, residual, True, False)
    return y if residual is None else (y, h)


def quantize_rows(x) -> RowsE4M3:
    """``x`` (..., C) as e4m3 rows with one scale each: activations between two products in 8 bits, or the rows of a weight
    (C_out, C_in) that is laid out once.  C <= 32768.  No gradient."""
    t = _row_type(x, "quantize_rows")
    if x.size(-1) > _MAX_NORM_C:
        raise ValueError(f"quantize_rows: rows of at most {_MAX_NORM_C} channels, got {x.size(-1)}")
    d = _device("quantize_rows", x)
    _no_grad_only("quantize_rows", x)
    x2, ldx = _rows2d(x)
    q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rows, C = x2.shape
    if rows:
        with _lib.device_ctx(d):
            rc = _lib.load().dgcn_quantize_rows_e4m3(x2.data_ptr(), ldx, t, q.data_ptr(), scale.data_ptr(), rows, C,
                                                     _lib.current_stream_handle(d))
        if rc:
            _lib.check(rc, "dgcn_quantize_rows_e4m3")
    return RowsE4M3(q, scale)


class RMSNorm(nn.Module):
    """``rms_norm_rows`` with its weight: ``norm_layer('rms', C)``.  ``forward(x, residual=None)`` returns ``y`` or
    ``(y, h)``; ``forward_e4m3`` the same in 8 bits."""

    def __init__(self, channels: int, eps: float = 1e-6):
        super().__init__()
        self.channels, self.eps = int(channels), float(eps)
        self.weight = nn.Parameter(torch.ones(self.channels))

    def forward(self, x, residual=None):
        return rms_norm_rows(x, self.weight, self.eps, residual)

    def forward_e4m3(self, x, residual=None):
        return rms_norm_rows_e4m3(x, self.weight, self.eps, residual)

    def extra_repr(self):
        return f"{self.channels}, eps={self.eps}"


# ---- product with epilogue ------------------------------------------------------------------------------------------
def _linear(x, weight, sx, sw, bias, residual, act: int, slope: float, in_type: int, out_dtype, keep: bool):
    """One call of checked arguments -> (y, what the backward keeps of the activation or None)."""
    lib = _lib.load()
    N, K = weight.shape
    y = x.new_empty((*x.shape[:-1], N), dtype=out_dtype)
    z = y.new_empty(y.shape) if keep and act != 0 else None
    if y.numel() == 0:
        return y, z
    x2, ldx = _rows2d(x)
    w2, ldw = _rows2d(weight)
    rows = x2.size(0)
    r2, ldr = (None, 0) if residual is None else _rows2d(residual)
    if bias is not None and not bias.is_contiguous():
        bias = bias.detach().contiguous()
    ptr = _lib.ptr
    px, pw = x2.data_ptr(), w2.data_ptr()
    # memory of this call alone, also inside a captured graph
    ws_bytes = lib.dgcn_linear_workspace(px, ldx, pw, ldw, in_type, rows, K, N)
    ws = y.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    d = y.get_device()
    with _lib.device_ctx(d):
        rc = lib.dgcn_linear_act(px, ldx, pw, ldw, ptr(sx), ptr(sw), ptr(bias),
                                 1 if bias is not None and bias.dtype == torch.float32 else 0, ptr(r2), ldr, act, slope, in_type,
                                 _TYPES[out_dtype], ptr(z), y.data_ptr(), rows, K, N, ptr(ws), ws_bytes,
                                 _lib.current_stream_handle(d))
    if rc:
        _lib.check(rc, "dgcn_linear_act")
    return y, z


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int, slope: float):
        y, z = _linear(x, weight, None, None, bias, residual, act, slope, _TYPES[x.dtype], x.dtype,
                       any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, z)
        ctx.cfg = (act, slope, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, z = ctx.saved_tensors
        act, slope, bias_type = ctx.cfg
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        gx = torch.zeros_like(x) if need_x and g.numel() == 0 else x.new_empty(x.shape) if need_x else None
        N, K = weight.shape
        if g.numel() == 0:                       # no rows: sums over nothing
            gw = weight.new_zeros((N, K)) if need_w else None
            gb = weight.new_zeros(N, dtype=bias_type) if need_b else None
            return gx, gw, gb, (g if need_r else None), None, None
        gw = weight.new_empty((N, K)) if need_w else None
        gb = weight.new_empty(N, dtype=bias_type) if need_b else None
        if need_x or need_w or need_b:
            lib = _lib.load()
            t = _TYPES[x.dtype]
            (x2, ldx), (w2, ldw), (g2, ldg) = _rows2d(x), _rows2d(weight), _rows2d(g)
            rows = g2.size(0)
            px, pw, pg, ptr = x2.data_ptr(), w2.data_ptr(), g2.data_ptr(), _lib.ptr
            ws_bytes = lib.dgcn_linear_bwd_workspace(pg, ldg, px, ldx, pw, ldw, act, t, need_x + 2 * need_w + 4 * need_b, rows,
                                                     K, N)
            ws = x.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
            d = g.get_device()
            with _lib.device_ctx(d):
                rc = lib.dgcn_linear_bwd(pg, ldg, px, ldx, pw, ldw, ptr(z), act, slope, t, ptr(gx), ptr(gw), ptr(gb),
                                         1 if bias_type == torch.float32 else 0, rows, K, N, ptr(ws), ws_bytes,
                                         _lib.current_stream_handle(d))
            if rc:
                _lib.check(rc, "dgcn_linear_bwd")
        return gx, gw, gb, (g if need_r else None), None, None


def _linear_checks(what, x, weight, bias, residual, act, out_dtype):
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"{what}: act must be one of {', '.join(ACTIVATIONS)}, got {act!r}")
    if weight.dim() != 2 or x.dim() < 1 or weight.size(1) != x.size(-1) or weight.size(0) < 1 or weight.size(1) < 1:
        raise ValueError(f"{what}: rows (..., K) and a weight (N, K) with K, N >= 1, got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    N, K = weight.shape
    if max(N, K) > _MAX_K:
        raise ValueError(f"{what}: at most {_MAX_K} channels, got {tuple(weight.shape)}")
    _param(bias, N, out_dtype, "bias")
    if residual is not None:
        _same_rows(residual, x, N, out_dtype, "residual")
    return code


def linear_act(x, weight, bias=None, act: str = "none", residual=None, neg_slope: float = 0.2):
    """``act(x @ weight.T + bias) + residual`` in one launch.

    ``x`` (..., K) and ``weight`` (N, K) in one of fp32, bf16, fp16; ``bias`` (N,) in that type or fp32; ``residual``
    (..., N) in that type; ``act`` one of :data:`ACTIVATIONS` (``neg_slope``: of leakyrelu, gelu: ``z Phi(z)``).  Gradients
    of all four; for them the forward keeps, where there is an activation, one value per result: the pre-activation of fp32
    rows, the activation's slope in 16-bit fixed point of 16-bit ones."""
    t = _row_type(x, "linear_act")
    if weight.dtype != x.dtype:
        raise TypeError(f"linear_act: weight must be {x.dtype} as the rows are, got {weight.dtype}")
    code = _linear_checks("linear_act", x, weight, bias, residual, act, x.dtype)
    _device("linear_act", x, weight, bias, residual)
    if _needs_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, code, neg_slope)
    return _linear(x, weight, None, None, bias, residual, code, neg_slope, t, x.dtype, False)[0]


def linear_act_e4m3(x: RowsE4M3, weight: RowsE4M3, bias=None, act: str = "none", residual=None,
                    out_dtype=torch.bfloat16, neg_slope: float = 0.2):
    """``act((x.data * x.scale) @ (weight.data * weight.scale).T + bias) + residual``: ``x`` rows (..., K), ``weight`` rows
    (N, K) (``quantize_rows`` of an nn.Linear weight, once); the result, ``residual`` and ``bias`` (or an fp32 bias) in
    ``out_dtype``; the scales join behind the sum.  For an fp32 result the products are summed in fp32; for a 16-bit one on
    the 8-bit matrix pipe at twice the rate, which cuts products that lie more than 2^13 below the largest of eight
    neighbouring ones (about 6e-5 of the result's root mean square over normal rows).  No gradient."""
    what = "linear_act_e4m3"
    if out_dtype not in _TYPES:
        raise TypeError(f"{what}: out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    (xd, sx), (wd, sw) = x, weight
    for name, r, s in (("x", xd, sx), ("weight", wd, sw)):
        if r.dtype != torch.float8_e4m3fn or s.dtype != torch.float32:
            raise TypeError(f"{what}: {name} must be float8_e4m3fn rows with float32 scales, got {r.dtype} and {s.dtype}")
        if s.shape != r.shape[:-1]:
            raise ValueError(f"{what}: {name} of shape {tuple(r.shape)} needs scales of shape {tuple(r.shape[:-1])}, got "
                             f"{tuple(s.shape)}")
    code = _linear_checks(what, xd, wd, bias, residual, act, out_dtype)
    _device(what, xd, sx, wd, sw, bias, residual)
    _no_grad_only(what, bias, residual, sx, sw)
    return _linear(xd, wd, sx.contiguous(), sw.contiguous(), bias, residual, code, neg_slope, _E4M3, out_dtype, False)[0]
