"""The operators of the node-wise MLP in 16, 32 and 8 bits, as cases to be measured.

Two sides give the same outputs for the same inputs: the plain form (``own`` false: elementary torch operations in 32
bits, rounded once at the end) and the package's kernels (``own`` true: ``deep_gcns_torch_amd.mlp_ops``).

    linear   y = act(x W^T + b) + r                       fp32 / bf16 / fp16, forward, or forward and backward
    norm     h = x + r,  y = h / rms(h) * w               fp32 / bf16 / fp16, forward, or forward and backward
    rows8    the same norm, or x alone, as e4m3 rows with one fp32 scale per row (scale = max|y| / 448)
    linear8  y = act(s_x s_w (q_x q_w^T) + b) + r         e4m3 rows times e4m3 weight rows, 16- or 32-bit result

A case is a dict: ``op``, ``dtype``, ``rows``, ``k`` (input channels), ``n`` (output channels; products only), ``act``,
``bias``, ``res`` (residual), ``norm`` (rows8 only) and ``train`` (gradients of every input are computed and returned).
"""
import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _case(name, op, dtype, rows, k, n=0, act="none", bias=False, res=False, norm=True, train=False):
    c = {"op": op, "dtype": dtype, "rows": rows, "k": k, "n": n, "act": act, "bias": bias, "res": res, "norm": norm,
         "train": train}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one row answered at a time: the weight's 33 MB are all there is to move
        _case("linear-1-row", "linear", "bf16", 1, 4096, 4096, "none", bias=True, res=True),
        # a ragged batch whose channels are multiples of nothing
        _case("linear-ragged", "linear", "fp16", 1021, 1013, 2047, "silu", bias=True),
        # a training step of the wide product of a transformer-sized MLP
        _case("linear-train-wide", "linear", "bf16", 8192, 4096, 16384, "gelu", bias=True, train=True),
        # a training step of GENConv's 128 -> 256 MLP stage over the ogbn-arxiv nodes, in the package's own type
        _case("linear-train-nodes", "linear", "fp32", 169343, 128, 256, "gelu", bias=True, train=True),
        # the norm in front of a layer, one row: latency
        _case("norm-1-row", "norm", "bf16", 1, 4096, res=True),
        # a training step of the residual sum and norm of a wide layer
        _case("norm-train-wide", "norm", "bf16", 16384, 4096, res=True, train=True),
        # the norm over the ogbn-arxiv nodes at 128 channels, in the package's own type
        _case("norm-train-nodes", "norm", "fp32", 169343, 128, train=True),
        # what a layer in 8 bits reads: the residual sum, normed and rounded to e4m3
        _case("rows8-norm-wide", "rows8", "bf16", 8192, 8192, res=True),
        # a few odd rows of it
        _case("rows8-norm-ragged", "rows8", "fp16", 7, 1001),
        # activations between two products in 8 bits, and a weight that is laid out once: no norm
        _case("rows8-wide", "rows8", "bf16", 8192, 16384, norm=False),
        # sixteen rows answered together in 8 bits
        _case("linear8-16-rows", "linear8", "bf16", 16, 4096, 16384, "silu", bias=True),
        # a long prompt, or all nodes of a graph, in 8 bits
        _case("linear8-wide", "linear8", "bf16", 8192, 8192, 8192, "none", bias=True, res=True),
    ]


MOST_FLOPS = 3 * 2 * 8192 * 4096 * 16384      # the wide training step's
MOST_VALUES = 8192 * 16384                    # the most values of one input or output of a listed case


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm; half of them rounded to what models use."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice([1, 1, 8, 64])
    return min(hi, max(lo, v if step == 1 or v < step else v // step * step))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "rows8", "linear8"])
    dtype = rng.choice(["bf16", "fp16", "fp32"] if op != "linear8" else ["bf16", "fp16", "bf16", "fp32"])
    train = op in ("linear", "norm") and rng.random() < 0.5
    rows = _spread(rng, 1, 200000)
    k = _spread(rng, 16, 16384)
    n = _spread(rng, 16, 16384) if op in ("linear", "linear8") else 0
    # gradients at the kink of relu and leakyrelu belong to whichever side rounding puts the value on: in 32 bits a
    # training case takes a smooth activation
    smooth = ["none", "gelu", "silu"]
    act = rng.choice(smooth if train and dtype == "fp32" else smooth + ["relu", "leakyrelu"]) if n else "none"
    passes = 3 if train else 1
    most = min(MOST_VALUES // max(k, n), MOST_FLOPS // max(1, 2 * passes * k * n)) if n else MOST_VALUES // k // passes
    if dtype == "fp32":
        most //= 4
    rows = max(1, min(rows, most))
    return _case(None, op, dtype, rows, k, n, act, bias=bool(n) and rng.random() < 0.7, res=rng.random() < 0.5,
                 norm=op != "rows8" or rng.random() < 0.6, train=train)


def work(case):
    r, k, n, b = case["rows"], case["k"], case["n"], BYTES[case["dtype"]]
    res, bias, train = case["res"], case["bias"], case["train"]
    if case["op"] == "linear":
        # forward: x, W, b, r in, y out; backward: g and the same inputs in, their gradients out
        fwd = r * k + n * k + n * bias + r * n * res + r * n
        bwd = (r * n + r * k + n * k + n * bias) if train else 0
        return {"bytes": b * (fwd + bwd), "flops": 2 * r * k * n * (3 if train else 1)}
    if case["op"] == "norm":
        fwd = r * k * (2 + 2 * res) + k                     # x [, r], w in; y [, h] out
        bwd = (r * k * (2 + res) + k) if train else 0       # g [, g_h] in; gx, gw out (the residual's gradient is gx)
        return {"bytes": b * (fwd + bwd), "flops": r * k * (16 if train else 5)}
    if case["op"] == "rows8":
        norm, res = case["norm"], res and case["norm"]
        return {"bytes": b * (r * k * (1 + 2 * res) + k * norm) + r * k + 4 * r, "flops": r * k * (7 if norm else 3)}
    # linear8: one byte a value, four a scale; bias and residual in the result's type
    return {"bytes": r * k + n * k + 4 * (r + n) + b * (n * bias + r * n * res + r * n), "flops": 2 * r * k * n}


def _randn(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * scale


def _plain_rows8(y):
    """Rows as e4m3 values and one fp32 scale each: scale = max|y| / 448, 1 for a row of zeros."""
    top = y.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, (top / E4M3_MAX).clamp_min(torch.finfo(torch.float32).tiny), torch.ones_like(top))
    return (y / scale).to(torch.float8_e4m3fn), scale.squeeze(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    t, r, k, n = TYPES[case["dtype"]], case["rows"], case["k"], case["n"]
    s = {"case": case}
    if case["op"] in ("linear", "linear8"):
        x, w = _randn(gen, r, k), _randn(gen, n, k, scale=k ** -0.5)
        s["bias"] = _randn(gen, n, scale=0.1).to(t) if case["bias"] else None
        s["res"] = _randn(gen, r, n).to(t) if case["res"] else None
        if case["op"] == "linear8":
            # what a model in 8 bits keeps: weight rows laid out once, and the rows that the norm handed on
            s["x"], s["w"] = _plain_rows8(x), _plain_rows8(w)
            return s
        s["x"], s["w"], width = x.to(t), w.to(t), n
    else:
        # residual streams have a few large channels
        x = _randn(gen, r, k) * (1.0 + 9.0 * (torch.rand(k, generator=gen, device="cuda") < 0.01))
        s["x"] = x.to(t)
        s["w"] = (1.0 + _randn(gen, k, scale=0.1)).to(t) if case["norm"] else None
        s["res"] = _randn(gen, r, k).to(t) if case["res"] and case["norm"] else None
        width = k
    if case["train"]:
        s["g"] = _randn(gen, r, width).to(t)
        s["gh"] = _randn(gen, r, width).to(t) if case["op"] == "norm" and case["res"] else None
        s["leaves"] = [s[name].requires_grad_() for name in ("x", "w", "bias", "res") if s.get(name) is not None]
    return s


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "leakyrelu":
        return torch.where(z > 0, z, 0.2 * z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _up(t, wide):
    return None if t is None else t.to(wide)


def _plain_linear(x, w, bias, res, act):
    z = x @ w.t()
    if bias is not None:
        z = z + bias
    y = _act(z, act)
    return y if res is None else y + res


def _plain_norm(x, w, res):
    h = x if res is None else x + res
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    return (y if w is None else y * w), h


def _plain(s):
    c, f = s["case"], torch.float32
    if c["op"] == "linear":
        return (_plain_linear(_up(s["x"], f), _up(s["w"], f), _up(s["bias"], f), _up(s["res"], f),
                              c["act"]).to(TYPES[c["dtype"]]),)
    if c["op"] == "linear8":
        (qx, sx), (qw, sw) = s["x"], s["w"]
        y = _plain_linear(qx.to(f) * sx[:, None], qw.to(f) * sw[:, None], _up(s["bias"], f), _up(s["res"], f), c["act"])
        return (y.to(TYPES[c["dtype"]]),)
    if c["op"] == "rows8" and not c["norm"]:
        return _plain_rows8(_up(s["x"], f))
    y, h = _plain_norm(_up(s["x"], f), _up(s["w"], f), _up(s["res"], f))
    h = (h.to(TYPES[c["dtype"]]),) if s["res"] is not None else ()
    return (_plain_rows8(y) if c["op"] == "rows8" else (y.to(TYPES[c["dtype"]]),)) + h


def _own(s):
    from deep_gcns_torch_amd import mlp_ops
    c = s["case"]
    if c["op"] == "linear":
        return (mlp_ops.linear_act(s["x"], s["w"], s["bias"], act=c["act"], residual=s["res"]),)
    if c["op"] == "linear8":
        x, w = mlp_ops.RowsE4M3(*s["x"]), mlp_ops.RowsE4M3(*s["w"])
        return (mlp_ops.linear_act_e4m3(x, w, s["bias"], act=c["act"], residual=s["res"], out_dtype=TYPES[c["dtype"]]),)
    if c["op"] == "rows8" and not c["norm"]:
        return tuple(mlp_ops.quantize_rows(s["x"]))
    fn = mlp_ops.rms_norm_rows_e4m3 if c["op"] == "rows8" else mlp_ops.rms_norm_rows
    out = fn(s["x"], s["w"], eps=EPS, residual=s["res"])
    y, h = (out, ()) if s["res"] is None else (out[0], (out[1],))
    return (tuple(y) if c["op"] == "rows8" else (y,)) + h


def run(state):
    out = _own(state) if own else _plain(state)
    if not state["case"]["train"]:
        return out
    ups = [state["g"]] + ([state["gh"]] if state["gh"] is not None else [])
    grads = torch.autograd.grad(out, state["leaves"], ups)
    return tuple(o.detach() for o in out) + tuple(grads)


def _gate(z, act):
    """(act(z), act'(z)) in 64 bits, written out."""
    if act == "relu":
        return torch.relu(z), (z > 0).double()
    if act == "leakyrelu":
        d = torch.full_like(z, 0.2)
        d[z > 0] = 1.0
        return z * d, d
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg * (1 + z * (1 - sg))
    return z, torch.ones_like(z)


def exact(case, seed):
    """What run() returns, before any rounding, in 64 bits."""
    with torch.no_grad():
        s = prepare(case, seed)
        s = {key: v.detach() if isinstance(v, torch.Tensor) else v for key, v in s.items()}
        d = torch.float64
        res = _up(s.get("res"), d)
        if case["op"] in ("linear", "linear8"):
            if case["op"] == "linear":
                x, w = s["x"].to(d), s["w"].to(d)
            else:
                x, w = (q.to(d).mul_(sc.to(d).unsqueeze(1)) for q, sc in (s["x"], s["w"]))
            z = torch.mm(x, w.mT)
            if s["bias"] is not None:
                z += s["bias"].to(d)
            y, slope = _gate(z, case["act"])
            if res is not None:
                y = y + res
            if not case["train"]:
                return (y,)
            g = s["g"].to(d)
            dz = g * slope
            out = [y, torch.mm(dz, w), torch.mm(dz.mT, x)]
            if s["bias"] is not None:
                out.append(dz.sum(0))
            return tuple(out + ([g] if res is not None else []))
        x = s["x"].to(d)
        w = s["w"].to(d) if s["w"] is not None else None
        h = x if res is None else x + res
        y = h
        if case["norm"]:
            inv = 1.0 / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / h.shape[1] + EPS)
            y = h * inv * w
        if case["op"] == "rows8":
            scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / E4M3_MAX
            scale[scale == 0] = 1.0
            return (y / scale.unsqueeze(1), scale) + ((h,) if res is not None else ())
        if not case["train"]:
            return (y,) + ((h,) if res is not None else ())
        g, unit = s["g"].to(d), h * inv
        gw = g * w
        gx = inv * (gw - unit * (gw * unit).mean(1, keepdim=True))
        if res is not None:
            gx = gx + s["gh"].to(d)
            return y, h, gx, (g * unit).sum(0), gx
        return y, gx, (g * unit).sum(0)
