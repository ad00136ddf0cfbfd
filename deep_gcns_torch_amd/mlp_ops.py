"""The node-wise MLP in 32, 16 and 8 bits: root-mean-square norm with the residual's addition, and the product with bias,
activation and residual in its epilogue (csrc/rms_norm.hip, csrc/linear_act.hip; csrc/mlp_host.cpp calls them).

``node_ops`` holds the fp32 row operators that the reference's own models use; these are the ones around them for models
whose rows are wider than 256 channels, or kept in bf16, fp16 or 8 bits (fp32 rows of at most 256 channels are ``node_ops``'s:
169,343 x 128 x 128 takes ``rows_linear`` 42 us and ``linear_act`` 58):

    h = x + r;  y = h * rsqrt(mean(h^2) + eps) * w     rms_norm_rows(x, w, eps, residual=r)        forward and backward
    the same y as e4m3 rows, one fp32 scale each       rms_norm_rows_e4m3(x, w, eps, residual=r)   forward
    x as e4m3 rows                                     quantize_rows(x)                            forward
    act(x W^T + b) + r                                 linear_act(x, W, b, act, residual=r)        forward and backward
    the same of e4m3 rows and an e4m3 weight           linear_act_e4m3(x, W, b, act, residual=r)   forward

Rows are the last dimension; leading dimensions are free and may be empty.  Sums and statistics are fp32, every result is
rounded once to its type.  Work runs on the current stream of the inputs' device; results do not depend on timing (no
atomics).  What an operator does not take raises, nothing falls back; so do forward-mode and second derivatives.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _lib

__all__ = ["ACTIVATIONS", "RMSNorm", "RowsE4M3", "linear_act", "linear_act_e4m3", "quantize_rows", "rms_norm_rows",
           "rms_norm_rows_e4m3"]

#: activation name -> code (include/dgcn.h)
ACTIVATIONS = {"none": 0, "relu": 1, "leakyrelu": 2, "gelu": 3, "silu": 4}
_ROW_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_MAX_NORM_C = 32768
_MAX_K = 1 << 20


class RowsE4M3(NamedTuple):
    """Rows in 8 bits: the row's values are ``data * scale``.  ``data`` (..., C) ``torch.float8_e4m3fn``, ``scale`` (...)
    fp32."""
    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        return (self.data.to(torch.float32) * self.scale.unsqueeze(-1)).to(dtype)


# Calls, allocation and autograd are C++ (csrc/mlp_host.cpp): a small call is bound by its host side.  It answers None where it
# does not take the arguments; the functions named _refuse_* then say why.
_host = None


def _native():
    """csrc/mlp_host.cpp, given the entry points of the loaded library.  Raises if it is not built."""
    global _host
    if _host is None:
        lib = _lib.load()
        try:
            from . import _mlp_host as host
        except ImportError as e:
            raise RuntimeError(f"deep_gcns_torch_amd/_mlp_host.so cannot be loaded ({e}): build it with "
                               "python -m deep_gcns_torch_amd.build") from e
        host.init({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in host.ENTRY_POINTS})
        _host = host
    return _host


def _refuse_rows(what: str, x: torch.Tensor, max_c=None) -> None:
    if x.dtype not in _ROW_TYPES:
        raise TypeError(f"{what}: rows must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError(f"{what}: rows need a last dimension of at least 1, got {tuple(x.shape)}")
    if max_c is not None and x.size(-1) > max_c:
        raise ValueError(f"{what}: rows of at most {max_c} channels, got {x.size(-1)}")


def _refuse_param(p, n: int, dtype, what: str) -> None:
    if p is None:
        return
    if p.dim() != 1 or p.size(0) != n:
        raise ValueError(f"{what} must have shape ({n},), got {tuple(p.shape)}")
    if p.dtype != dtype and p.dtype != torch.float32:
        raise TypeError(f"{what} must be {dtype} or float32, got {p.dtype}")


def _refuse_residual(r, x: torch.Tensor, n: int, dtype) -> None:
    if r is None:
        return
    want = (*x.shape[:-1], n)
    if r.shape != want:
        raise ValueError(f"residual must have shape {tuple(want)}, got {tuple(r.shape)}")
    if r.dtype != dtype:
        raise TypeError(f"residual must be {dtype}, got {r.dtype}")


def _refuse_rest(what: str, tensors, no_grad=False):
    """The checks common to all, and the end of a refusal: always raises."""
    _lib.require_device(*tensors)                # raises: a CPU tensor, or two devices
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative")
    if no_grad and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or on tensors that require none")
    raise RuntimeError(f"{what} does not take these arguments")


# ---- root-mean-square norm ------------------------------------------------------------------------------------------
def _refuse_rms(what, x, weight, residual, no_grad):
    _refuse_rows(what, x, _MAX_NORM_C)
    _refuse_param(weight, x.size(-1), x.dtype, "weight")
    _refuse_residual(residual, x, x.size(-1), x.dtype)
    _refuse_rest(what, (x, weight, residual), no_grad)


def rms_norm_rows(x, weight=None, eps: float = 1e-6, residual=None):
    """``h = x [+ residual]``, ``y = h * rsqrt(mean(h^2) + eps) [* weight]`` over the last dimension.

    Returns ``y``, or ``(y, h)`` with a residual: ``h`` is the stream that the next layer adds to.  ``x`` (..., C) fp32,
    bf16 or fp16, C <= 32768; ``residual`` of the same shape and type; ``weight`` (C,) in the rows' type or fp32.  ``y`` and its
    gradient (of x, weight and residual) are those of the fp32 sum: the backward keeps ``x`` and ``residual``, not ``h``."""
    out = (_host or _native()).rms_norm(x, weight, eps, residual)
    return out if out is not None else _refuse_rms("rms_norm_rows", x, weight, residual, False)


def rms_norm_rows_e4m3(x, weight=None, eps: float = 1e-6, residual=None):
    """``rms_norm_rows`` whose ``y`` leaves as :class:`RowsE4M3`: ``scale = max|y| / 448`` per row (1 for a row of zeros).
    Returns the rows, or ``(rows, h)`` with a residual.  A NaN or an infinity becomes NaN in its own place.  No gradient."""
    out = (_host or _native()).rms_norm_e4m3(x, weight, eps, residual)
    if out is None:
        _refuse_rms("rms_norm_rows_e4m3", x, weight, residual, True)
    return RowsE4M3(*out) if residual is None else (RowsE4M3(out[0], out[1]), out[2])


def quantize_rows(x) -> RowsE4M3:
    """``x`` (..., C) as e4m3 rows with one scale each: activations between two products in 8 bits, or the rows of a weight
    (C_out, C_in) that is laid out once.  C <= 32768.  No gradient."""
    out = (_host or _native()).quantize_rows(x)
    if out is None:
        _refuse_rows("quantize_rows", x, _MAX_NORM_C)
        _refuse_rest("quantize_rows", (x,), True)
    return RowsE4M3(*out)


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
def _refuse_linear(what, x, weight, bias, residual, out_dtype):
    if weight.dim() != 2 or x.dim() < 1 or weight.size(1) != x.size(-1) or weight.size(0) < 1 or weight.size(1) < 1:
        raise ValueError(f"{what}: rows (..., K) and a weight (N, K) with K, N >= 1, got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    if max(weight.shape) > _MAX_K:
        raise ValueError(f"{what}: at most {_MAX_K} channels, got {tuple(weight.shape)}")
    _refuse_param(bias, weight.size(0), out_dtype, "bias")
    _refuse_residual(residual, x, weight.size(0), out_dtype)


def _act_code(what: str, act: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"{what}: act must be one of {', '.join(ACTIVATIONS)}, got {act!r}")
    return code


def linear_act(x, weight, bias=None, act: str = "none", residual=None, neg_slope: float = 0.2):
    """``act(x @ weight.T + bias) + residual``, all of it in the product's launch (a reduction that is split ends in a second one;
    rows that do not start on dwords are copied first, but for the few that are read in place).

    ``x`` (..., K) and ``weight`` (N, K) in one of fp32, bf16, fp16; ``bias`` (N,) in that type or fp32; ``residual``
    (..., N) in that type; ``act`` one of :data:`ACTIVATIONS` (``neg_slope``: of leakyrelu, gelu: ``z Phi(z)``).  Gradients
    of all four; for them the forward keeps, where there is an activation, one value per result: the pre-activation of fp32
    rows, the activation's slope as a 16-bit code of 16-bit ones (within 2^-16, and within 2^-10 of itself where a unit is
    saturated, from -2^-6 to -2^-45; what is smaller is 0).  Of 16-bit rows the gradient of the pre-activation is rounded to
    their type before its two products.  Infinities and NaN give what the products give, in every type."""
    code = _act_code("linear_act", act)
    y = (_host or _native()).linear_act(x, weight, bias, code, residual, neg_slope)
    if y is None:
        _refuse_rows("linear_act", x)
        if weight.dtype != x.dtype:
            raise TypeError(f"linear_act: weight must be {x.dtype} as the rows are, got {weight.dtype}")
        _refuse_linear("linear_act", x, weight, bias, residual, x.dtype)
        _refuse_rest("linear_act", (x, weight, bias, residual))
    return y


def linear_act_e4m3(x: RowsE4M3, weight: RowsE4M3, bias=None, act: str = "none", residual=None,
                    out_dtype=torch.bfloat16, neg_slope: float = 0.2):
    """``act((x.data * x.scale) @ (weight.data * weight.scale).T + bias) + residual``: ``x`` rows (..., K), ``weight`` rows
    (N, K) (``quantize_rows`` of an nn.Linear weight, once); the result, ``residual`` and ``bias`` (or an fp32 bias) in
    ``out_dtype``; the scales join behind the sum.  For an fp32 result, and for up to 16 rows (but
    where few channels meet a long K), the products are summed in fp32; for a 16-bit one of more rows on the 8-bit matrix
    pipe at twice the rate, which cuts products that lie more than 2^13 below the largest of eight neighbouring ones (about
    6e-5 of the result's root mean square over normal rows).  No gradient."""
    what = "linear_act_e4m3"
    if out_dtype not in _ROW_TYPES:
        raise TypeError(f"{what}: out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    code = _act_code(what, act)
    (xd, sx), (wd, sw) = x, weight
    y = (_host or _native()).linear_act_e4m3(xd, sx, wd, sw, bias, code, residual, out_dtype, neg_slope)
    if y is None:
        for name, r, s in (("x", xd, sx), ("weight", wd, sw)):
            if r.dtype != torch.float8_e4m3fn or s.dtype != torch.float32:
                raise TypeError(f"{what}: {name} must be float8_e4m3fn rows with float32 scales, got {r.dtype} and {s.dtype}")
            if s.shape != r.shape[:-1]:
                raise ValueError(f"{what}: {name} of shape {tuple(r.shape)} needs scales of shape {tuple(r.shape[:-1])}, got "
                                 f"{tuple(s.shape)}")
        _refuse_linear(what, xd, wd, bias, residual, out_dtype)
        _refuse_rest(what, (xd, sx, wd, sw, bias, residual), True)
    return y
