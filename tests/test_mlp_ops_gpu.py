"""mlp_ops on the device against a plain implementation in 64 bits.

Tolerances are bounds, element by element, counted from the operators' roundings before the first run: a sum of n fp32
terms is off by at most n 2^-24 of the sum of their magnitudes, a result by half a step of its type, the stored
pre-activation z and the stored h by half a step of theirs.  u below is 2^-24."""
import math

import pytest
import torch

from deep_gcns_torch_amd import blocks, mlp_ops
from deep_gcns_torch_amd.mlp_ops import RowsE4M3

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # least subnormal
# largest |act'| and |act''| (gelu: 1.13, 0.8; silu: 1.1, 0.5), rounded up
LIP = {"none": (1.0, 0.0), "relu": (1.0, 0.0), "leakyrelu": (1.0, 0.0), "gelu": (1.13, 0.8), "silu": (1.1, 0.5)}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(*shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def within(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got.double()).all(), what
    far = ((got.double() - want).abs() - bound).max().item() if got.numel() else 0.0
    assert far <= 0, f"{what}: {far:.3e} over its bound"


# ---- norm -----------------------------------------------------------------------------------------------------------
def norm_ref(x, w, r, eps):
    h = x.double() if r is None else x.double() + r.double()
    rstd = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h, rstd, h * rstd * (1.0 if w is None else w.double())


def y_bound(y, C, dtype):
    """x + r: u; the mean of squares: (C + 3) u, half of it in rstd; sqrt, quotient, two products: 6 u."""
    return y.abs() * ((C + 3) / 2 + 7) * U + y.abs() * half_step(dtype) * 1.01 + TINY[dtype]


NORM_SHAPES = [(1, 4096), (1, 1), (3, 7), (5, 16), (257, 33), (64, 128), (9, 255), (130, 513), (3, 1001), (2, 2049),
               (17, 4096), (3, 8191), (2, 16384), (2, 32768), (0, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, C", NORM_SHAPES)
@pytest.mark.parametrize("weight, residual", [("same", True), ("fp32", False), (None, True)])
def test_norm(dtype, rows, C, weight, residual):
    x = rand(rows, C, dtype=dtype, seed=1).requires_grad_()
    r = rand(rows, C, dtype=dtype, seed=2).requires_grad_() if residual else None
    w = None
    if weight:
        w = (1 + rand(C, dtype=torch.float32, seed=3, scale=0.3)).to(dtype if weight == "same" else torch.float32)
        w.requires_grad_()
    g, gh = rand(rows, C, dtype=dtype, seed=4), rand(rows, C, dtype=dtype, seed=5)
    out = mlp_ops.rms_norm_rows(x, w, eps=1e-5, residual=r)
    y, h = out if residual else (out, None)
    with torch.no_grad():
        plain = mlp_ops.rms_norm_rows(x, w, eps=1e-5, residual=r)
    assert torch.equal(plain[0] if residual else plain, y)
    h64, rstd, y64 = norm_ref(x, w, r, 1e-5)
    within(y, y64, y_bound(y64, C, dtype), "y")
    if residual:
        within(h, h64, h64.abs() * (half_step(dtype) * 1.01 + U) + TINY[dtype], "h")
    leaves = [t for t in (x, w, r) if t is not None]
    grads = torch.autograd.grad((y, h) if residual else y, leaves, (g, gh) if residual else g)
    eh = half_step(dtype) if residual else 0.0                      # the stored h
    w64 = torch.ones(C, device="cuda", dtype=torch.float64) if w is None else w.detach().double()
    g64, xh = g.double(), h64 * rstd
    gw = g64 * w64
    dot = (gw * xh).mean(-1, keepdim=True)
    dx = rstd * (gw - xh * dot) + (gh.double() if residual else 0.0)
    rel = (C + 20) * U
    edot = (gw * xh).abs().mean(-1, keepdim=True) * (eh * 1.01 + rel)
    edx = rstd * (xh.abs() * edot + (xh * dot).abs() * (eh * 1.01 + rel) + gw.abs() * rel) + (rstd * (gw.abs() + (xh * dot).abs())) * 8 * U
    edx = edx + dx.abs() * (half_step(dtype) * 1.01 + 2 * U) + TINY[dtype] + (gh.double().abs() * 2 * U if residual else 0.0)
    within(grads[0], dx, edx, "gx")
    if residual:
        within(grads[-1], dx, edx, "gr")
    if w is not None:
        gw64 = (g64 * xh).sum(0)
        egw = (g64 * xh).abs().sum(0) * (eh * 1.01 + (rows + C + 20) * U) + gw64.abs() * half_step(w.dtype) * 1.01 + TINY[w.dtype]
        within(grads[1], gw64, egw, "gw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, C", NORM_SHAPES)
@pytest.mark.parametrize("kind", ["norm", "norm+res", "rows"])
def test_rows_e4m3(dtype, rows, C, kind):
    x = rand(rows, C, dtype=dtype, seed=1, scale=3.0)
    w = (1 + rand(C, dtype=torch.float32, seed=3, scale=0.3)).to(dtype)
    r = rand(rows, C, dtype=dtype, seed=2) if kind == "norm+res" else None
    if kind == "rows":
        q, y64, rel = mlp_ops.quantize_rows(x), x.double(), 0.0
    else:
        out = mlp_ops.rms_norm_rows_e4m3(x, w, eps=1e-5, residual=r)
        q, h = out if r is not None else (out, None)
        h64, _, y64 = norm_ref(x, w, r, 1e-5)
        rel = ((C + 3) / 2 + 7) * U
        if r is not None:
            assert torch.equal(h, (x.float() + r.float()).to(dtype))
    assert q.data.dtype == torch.float8_e4m3fn and q.data.shape == x.shape and q.scale.shape == x.shape[:-1]
    if rows == 0:
        return
    top = y64.abs().amax(-1)
    within(q.scale, top / 448, top / 448 * (rel + 4 * U), "scale")
    # three mantissa bits: half a step is 2^-4 of the value, and 2^-10 below the least normal 2^-6 (both times the scale)
    bound = y64.abs() * (2.0 ** -4 + 2 * rel + 8 * U) + q.scale.double().unsqueeze(-1) * 2.0 ** -10 * (1 + 1e-5)
    within(q.data.double() * q.scale.double().unsqueeze(-1), y64, bound, "q * scale")
    assert (q.data.float().abs().amax(-1) == 448).all()
    assert torch.equal(q.dequantize(), q.data.float() * q.scale.unsqueeze(-1))


def test_rows_e4m3_values():
    """Every e4m3 number is its own rounding; ties go to even; what is not finite stays in its place."""
    code = torch.arange(256, device="cuda", dtype=torch.uint8)
    v = code.view(torch.float8_e4m3fn).float()
    v = v[torch.isfinite(v)]                                        # 254 values, largest 448: the scale is 1
    q = mlp_ops.quantize_rows(v.view(1, -1))
    assert q.scale.item() == 1.0 and torch.equal(q.data.float().view(-1), v)
    pos = v[v >= 0].unique()
    mid = (pos[:-1] + pos[1:]) / 2                                  # exact in fp32
    row = torch.cat([mid, torch.tensor([448.0], device="cuda")]).view(1, -1)
    got = mlp_ops.quantize_rows(row).data[0, :-1]
    assert (got.view(torch.uint8) % 2 == 0).all()                   # the neighbour whose last bit is 0
    assert ((got.float() == pos[:-1]) | (got.float() == pos[1:])).all()
    bad = torch.tensor([[1.0, float("nan"), -2.0, float("inf")], [0.0, 0.0, -0.0, 0.0],
                        [float("nan")] * 4, [1e-44, 0.0, 0.0, -1e-44]], device="cuda")
    q = mlp_ops.quantize_rows(bad)
    d = q.data.float()
    assert torch.allclose(q.scale[0], torch.tensor(2 / 448, device="cuda")) and q.scale[1] == 1 and q.scale[2] == 1
    assert q.scale[3] == torch.finfo(torch.float32).tiny
    assert torch.isnan(d[0]).tolist() == [False, True, False, True] and d[0, 2] == -448 and d[0, 0] == 224
    assert (d[1] == 0).all() and torch.isnan(d[2]).all() and (d[3] == 0).all()


# ---- product --------------------------------------------------------------------------------------------------------
def act_ref(z, act, slope=0.2):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "leakyrelu":
        return torch.where(z > 0, z, slope * z), torch.where(z > 0, 1.0, slope).double()
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def terms(K, dtype):
    """Roundings of a sum of K products, in u: 16- and 8-bit products are exact in fp32; an fp32 one may be six products
    of bf16 parts, of which three parts of 2^-24 are dropped."""
    return 6 * K + 12 if dtype == torch.float32 else K + 4


def linear_bounds(x, w, b, act, dtype, in_dtype=None):
    """(z, bound of the fp32 z, bound of act(z)) in 64 bits."""
    x64, w64 = x.double(), w.double()
    z, mag = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    ez = mag * terms(x.size(-1), in_dtype or dtype) * U
    y, _ = act_ref(z, act)
    # act(z) itself: a few roundings and a base-2 exponential (|z| 2^-24 in its argument); for 16-bit results a quarter
    # of half a step more, for whatever is used for the distribution function
    ea = y.abs() * (16 + 4 * z.abs()) * U + (0.25 * half_step(dtype) * y.abs() if dtype != torch.float32 else 0.0)
    if act in ("none", "relu", "leakyrelu"):
        ea = y.abs() * 2 * U
    return z, ez, y, LIP[act][0] * ez + ea


def check_linear(x, w, b, r, act, y, dtype):
    z, ez, y64, ey = linear_bounds(x, w, b, act, dtype)
    if r is not None:
        y64 = y64 + r.double()
    within(y, y64, ey * 1.01 + y64.abs() * (half_step(dtype) * 1.01 + U) + TINY[dtype], "y")
    return z, ez


def check_linear_grads(x, w, b, r, act, g, grads, z, ez, dtype):
    g64, (_, slope) = g.double(), act_ref(z, act)
    dz = g64 * slope
    keep = half_step(dtype)                                         # z is stored in the rows' type
    ed = torch.zeros_like(dz)
    if act != "none":
        ezs = ez + z.abs() * keep * 1.01 + TINY[dtype]
        ed = g64.abs() * (LIP[act][1] * ezs + 24 * U + (0.25 * keep if dtype != torch.float32 else 0)) + dz.abs() * (keep * 1.01 + 4 * U)
        if act in ("relu", "leakyrelu"):
            ed = ed + g64.abs() * (z.abs() <= ezs)                  # the kink may fall to either side
    x64, w64, rows, N = x.double(), w.double(), x.size(0), w.size(0)
    dx, dw = dz @ w64, dz.t() @ x64
    adz = dz.abs() + ed
    bx = ed @ w64.abs() + (adz @ w64.abs()) * terms(N, dtype) * U + dx.abs() * keep * 1.01 + TINY[dtype]
    bw = ed.t() @ x64.abs() + (adz.t() @ x64.abs()) * terms(rows, dtype) * U + dw.abs() * keep * 1.01 + TINY[dtype]
    within(grads[0], dx, bx, "gx")
    within(grads[1], dw, bw, "gw")
    at = 2
    if b is not None:
        db = dz.sum(0)
        within(grads[at], db, ed.sum(0) + adz.sum(0) * (rows + 4) * U + db.abs() * half_step(b.dtype) * 1.01 + TINY[b.dtype], "gb")
        at += 1
    if r is not None:
        assert torch.equal(grads[at], g)


LINEAR_SHAPES = [(1, 8, 8), (1, 1, 1), (1, 4096, 512), (2, 17, 5), (16, 256, 4096), (17, 129, 65), (33, 64, 300),
                 (65, 1000, 72), (128, 128, 128), (100, 2048, 40), (257, 520, 264), (300, 96, 1025), (1500, 112, 224),
                 (5000, 128, 256), (1025, 13, 7), (0, 16, 24),
                 # whole and ragged tiles of each size, long and split reductions
                 (4096, 72, 4104), (2049, 1096, 2056), (60, 8192, 512), (700, 4096, 264), (129, 6152, 136), (9000, 264, 520),
                 # few rows: one to four tiles of 16, rows that end inside a step, channels that end inside 16
                 (15, 4095, 33), (32, 1030, 100), (47, 777, 1000), (64, 2048, 130), (5, 70, 4100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, K, N", LINEAR_SHAPES)
@pytest.mark.parametrize("act, bias, residual", [("none", None, False), ("gelu", "same", True), ("relu", "fp32", False),
                                                 ("silu", "same", False), ("leakyrelu", None, True)])
def test_linear_act(dtype, rows, K, N, act, bias, residual):
    x = rand(rows, K, dtype=dtype, seed=1).requires_grad_()
    w = rand(N, K, dtype=dtype, seed=2, scale=K ** -0.5).requires_grad_()
    b = rand(N, dtype=dtype if bias == "same" else torch.float32, seed=3).requires_grad_() if bias else None
    r = rand(rows, N, dtype=dtype, seed=4).requires_grad_() if residual else None
    g = rand(rows, N, dtype=dtype, seed=5)
    y = mlp_ops.linear_act(x, w, b, act=act, residual=r)
    with torch.no_grad():
        assert torch.equal(mlp_ops.linear_act(x, w, b, act=act, residual=r), y)
    grads = torch.autograd.grad(y, [t for t in (x, w, b, r) if t is not None], g)
    with torch.no_grad():
        z, ez = check_linear(x, w, b, r, act, y, dtype)
        check_linear_grads(x, w, b, r, act, g, grads, z, ez, dtype)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("rows, K, N", LINEAR_SHAPES)
@pytest.mark.parametrize("act, bias, residual", [("none", "fp32", True), ("silu", "same", False)])
def test_linear_act_e4m3(out, rows, K, N, act, bias, residual):
    x = mlp_ops.quantize_rows(rand(rows, K, dtype=torch.float32, seed=1))
    w = mlp_ops.quantize_rows(rand(N, K, dtype=torch.float32, seed=2, scale=K ** -0.5))
    b = rand(N, dtype=out if bias == "same" else torch.float32, seed=3)
    r = rand(rows, N, dtype=out, seed=4) if residual else None
    y = mlp_ops.linear_act_e4m3(x, w, b, act=act, residual=r, out_dtype=out)
    xd, wd = (t.data.double() * t.scale.double().unsqueeze(-1) for t in (x, w))
    z, ez, y64, ey = linear_bounds(xd, wd, b, act, out, torch.float8_e4m3fn)
    if out != torch.float32:
        # The 8-bit matrix instruction cuts each product to a multiple of 2^(E - 13), E the exponent of the largest of the
        # eight neighbouring ones (test_e4m3_products_share_an_exponent_by_eight): seven products of each eight are off by
        # less than 2^-13 of the largest, which is at most max|x| max|w| over the eight.
        top = [torch.nn.functional.pad(t.abs(), (0, -K % 8)).unflatten(1, (-1, 8)).amax(-1) for t in (xd, wd)]
        ey = ey + LIP[act][0] * 7 * 2.0 ** -13 * (top[0] @ top[1].t())
    y64 = y64 if r is None else y64 + r.double()
    within(y, y64, ey * 1.01 + z.abs() * 4 * U + y64.abs() * (half_step(out) * 1.01 + U) + TINY[out], "y")


def test_e4m3_products_share_an_exponent_by_eight():
    """What the tolerance above says of the instruction, and that an fp32 result does not have it: 2^16 - 2^16 + 2^(16 - d)."""
    for where, d, kept in ((2, 13, True), (2, 14, False), (7, 14, False), (8, 20, True), (40, 26, True)):
        x, w = torch.zeros(64, 128, device="cuda"), torch.zeros(64, 128, device="cuda")
        x[:, 0], w[:, 0], x[:, 1], w[:, 1] = 256.0, 256.0, 256.0, -256.0
        x[:, where], w[:, where] = 2.0 ** ((17 - d) // 2), 2.0 ** (16 - d - (17 - d) // 2)
        one = torch.ones(64, device="cuda")
        rows = [RowsE4M3(t.to(torch.float8_e4m3fn), one) for t in (x, w)]
        full = torch.full((64, 64), 2.0 ** (16 - d), device="cuda")
        assert torch.equal(mlp_ops.linear_act_e4m3(*rows, out_dtype=torch.float32), full)
        assert torch.equal(mlp_ops.linear_act_e4m3(*rows, out_dtype=torch.bfloat16).float(), full if kept else 0 * full)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_leading_dimensions(dtype):
    """Rows with a stride, rows that repeat, columns of a wider matrix, a transposed weight, a misaligned start."""
    big = rand(40, 3, 100, dtype=dtype, seed=1)
    x, w0 = big[:, 1, 3:70], rand(70, 90, dtype=dtype, seed=2, scale=0.1)
    assert x.stride() == (300, 1)
    for w in (w0[:, 11:78], rand(67, 50, dtype=dtype, seed=3, scale=0.1).t()):
        r = rand(w.size(0), dtype=dtype, seed=4).expand(40, -1)
        y = mlp_ops.linear_act(x, w, act="silu", residual=r)
        assert torch.equal(y, mlp_ops.linear_act(x.clone(), w.clone(), act="silu", residual=r.clone()))
        check_linear(x, w, None, r, "silu", y, dtype)
    y3 = mlp_ops.linear_act(big[..., :64], w0[:, :64])
    assert y3.shape == (40, 3, 70) and torch.equal(y3.view(120, 70), mlp_ops.linear_act(big[..., :64].reshape(120, 64), w0[:, :64].contiguous()))
    one = mlp_ops.linear_act(big[0, 0, :90], w0)
    assert one.shape == (70,) and torch.equal(one, mlp_ops.linear_act(big[0, :1, :90], w0)[0])
    y, h = mlp_ops.rms_norm_rows(big[:, 1, 3:70], residual=rand(67, dtype=dtype, seed=5).expand(40, 67))
    y2, h2 = mlp_ops.rms_norm_rows(x.clone(), residual=rand(67, dtype=dtype, seed=5).repeat(40, 1))
    assert torch.equal(y, y2) and torch.equal(h, h2)
    q, q2 = mlp_ops.quantize_rows(big[:, 1, 3:70]), mlp_ops.quantize_rows(x.clone())
    assert torch.equal(q.data.view(torch.uint8), q2.data.view(torch.uint8)) and torch.equal(q.scale, q2.scale)
    # 8-bit rows: every second row of a wider buffer, from an odd byte on
    buf = mlp_ops.quantize_rows(rand(80, 101, dtype=dtype, seed=6))
    xs = RowsE4M3(buf.data[::2, 5:94], buf.scale[::2])
    ws = RowsE4M3(buf.data[1:60, 7:96], buf.scale[1:60])
    xc, wc = (RowsE4M3(t.data.view(torch.uint8).clone().view(torch.float8_e4m3fn), t.scale.clone()) for t in (xs, ws))
    assert torch.equal(mlp_ops.linear_act_e4m3(xs, ws, out_dtype=dtype), mlp_ops.linear_act_e4m3(xc, wc, out_dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [1, 2, 6, 30, 33, 62, 66, 90, 127, 130, 190])
def test_rows_that_end_inside_a_chunk_see_nothing_behind(dtype, K):
    """Rows of a wider matrix whose neighbours are NaN and infinite: nothing behind K, and nothing of another row, gets in."""
    big = torch.full((200, 200), float("nan"), device="cuda", dtype=dtype)
    big[:, 150:] = float("inf")
    wide = big.clone()
    big[:, :K] = rand(200, K, dtype=dtype, seed=1)
    wide[:, :K] = rand(200, K, dtype=dtype, seed=2, scale=0.2)
    x, w = big[:, :K], wide[:, :K]
    y = mlp_ops.linear_act(x, w)
    assert torch.isfinite(y).all() and torch.equal(y, mlp_ops.linear_act(x.contiguous(), w.contiguous()))
    check_linear(x, w, None, None, "none", y, dtype)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    g = big[:, :200].clone()
    g[:, K:] = 0
    g = torch.cat([g[:, :K], torch.zeros(200, 200 - K, device="cuda", dtype=dtype)], 1)
    g2 = torch.full((200, 260), float("nan"), device="cuda", dtype=dtype)
    g2[:, 3:203] = g
    for grad in (g, g2[:, 3:203]):
        gx, gw = torch.autograd.grad(mlp_ops.linear_act(xg, wg), (xg, wg), grad)
        z, ez, _, _ = linear_bounds(xg.detach(), wg.detach(), None, "none", dtype)
        check_linear_grads(xg.detach(), wg.detach(), None, None, "none", g, (gx, gw), z, ez, dtype)
    q = mlp_ops.quantize_rows(x.contiguous())
    nan = torch.full((200, 200), 0x7f, device="cuda", dtype=torch.uint8)
    nan[:, :K] = q.data.view(torch.uint8)
    part = RowsE4M3(nan.view(torch.float8_e4m3fn)[:, :K], q.scale)
    assert torch.equal(mlp_ops.linear_act_e4m3(part, part, out_dtype=dtype), mlp_ops.linear_act_e4m3(q, q, out_dtype=dtype))


def test_gradients_of_strided_and_broadcast_inputs():
    x0 = rand(50, 40, dtype=torch.float32, seed=1).requires_grad_()
    w = rand(24, 20, dtype=torch.float32, seed=2, scale=0.2).requires_grad_()
    r = rand(24, dtype=torch.float32, seed=3).requires_grad_()
    y = mlp_ops.linear_act(x0[:, 7:27], w, act="silu", residual=r.expand(50, 24))
    g = torch.ones((), device="cuda").expand(50, 24)                    # the gradient of y.sum(): strides (0, 0)
    gx, gw, gr = torch.autograd.grad(y, (x0, w, r), g)
    x, z = x0.detach()[:, 7:27].double(), x0.detach()[:, 7:27].double() @ w.detach().double().t()
    dz = act_ref(z, "silu")[1]
    assert (gx[:, :7] == 0).all() and (gx[:, 27:] == 0).all()
    torch.testing.assert_close(gx[:, 7:27].double(), dz @ w.detach().double(), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(gw.double(), dz.t() @ x, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(gr, torch.full_like(gr, 50.0))
    # the sum alone is used, or the normed rows alone
    h0 = rand(6, 33, dtype=torch.float32, seed=4).requires_grad_()
    y, h = mlp_ops.rms_norm_rows(h0, residual=h0)
    assert torch.equal(torch.autograd.grad(h.sum(), h0, retain_graph=True)[0], torch.full_like(h0, 2.0))
    gy, = torch.autograd.grad(y, h0, rand(6, 33, dtype=torch.float32, seed=5))
    assert torch.isfinite(gy).all() and gy.abs().max() > 0
    with pytest.raises(RuntimeError, match="has no gradient"):
        mlp_ops.quantize_rows(h0)
    with pytest.raises(RuntimeError, match="has no gradient"):
        mlp_ops.rms_norm_rows_e4m3(h0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 70, 200])
def test_gradients_of_rows_that_repeat_or_overlap(dtype, rows):
    """One row expanded over all, windows of a line that overlap, a weight likewise, and a gradient that is one row expanded
    (of y.sum(0)): sums over `rows` rows, not over a tile's."""
    row, line = rand(36, dtype=dtype, seed=1), rand(4 * rows + 100, dtype=dtype, seed=2)
    wline, grow = rand(400, dtype=dtype, seed=3, scale=0.2), rand(24, dtype=dtype, seed=4)
    w = wline.as_strided((24, 36), (8, 1))
    for x in (row.expand(rows, 36), line.as_strided((rows, 36), (4, 1))):
        xg, wg = x.detach().requires_grad_(), w.detach().requires_grad_()
        b = torch.zeros(24, device="cuda", dtype=dtype).requires_grad_()
        assert xg.stride(0) in (0, 4) and wg.stride(0) == 8
        for bias in (None, b):
            y = mlp_ops.linear_act(xg, wg, bias)
            g = grow.expand(rows, 24)
            grads = torch.autograd.grad(y, [t for t in (xg, wg, bias) if t is not None], g)
            z, ez = check_linear(x, w, None if bias is None else b.detach(), None, "none", y.detach(), dtype)
            check_linear_grads(x, w, None if bias is None else b.detach(), None, "none", g, grads, z, ez, dtype)


def test_gradients_against_differences():
    """<grad, v> against (f(x + s v) - f(x - s v)) / 2 s, f = <y, g> summed in 64 bits, s a power of two.  Bound: what the
    same difference of the 64-bit reference is off by (truncation), and twice the outputs' bound over 2 s."""
    s = 2.0 ** -7
    x, w, b = (rand(*sh, dtype=torch.float32, seed=i, scale=sc) for i, (sh, sc) in
               enumerate([((30, 48), 1.0), ((20, 48), 0.15), ((20,), 0.3)]))
    g = rand(30, 20, dtype=torch.float32, seed=7)
    for act in ("gelu", "silu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(mlp_ops.linear_act(*leaves, act=act), leaves, g)
        for k in range(3):
            v = rand(*leaves[k].shape, dtype=torch.float32, seed=20 + k)
            sides, sides64, room = [], [], 0.0
            for sign in (s, -s):
                args = [t.clone() for t in (x, w, b)]
                args[k] = args[k] + sign * v
                sides.append((mlp_ops.linear_act(*args, act=act).double() * g.double()).sum())
                _, _, y64, ey = linear_bounds(*args, act, torch.float32)
                sides64.append((y64 * g.double()).sum())
                room += ((ey + y64.abs() * 2 * U) * g.double().abs()).sum().item() / (2 * s)
            a64 = [t.double().requires_grad_() for t in (x, w, b)]
            z64 = a64[0] @ a64[1].t() + a64[2]
            y64 = z64 * torch.sigmoid(z64) if act == "silu" else z64 * 0.5 * torch.erfc(-z64 / math.sqrt(2))
            exact = (torch.autograd.grad(y64, a64[k], g.double())[0] * v.double()).sum()
            trunc = ((sides64[0] - sides64[1]) / (2 * s) - exact).abs().item()
            got, diff = (grads[k].double() * v.double()).sum(), (sides[0] - sides[1]) / (2 * s)
            assert (got - diff).abs().item() <= room + trunc + 1e-4 * exact.abs().item() + 1e-4, (act, k)


def test_not_finite_rows_stay_in_their_rows():
    x, w = rand(70, 96, dtype=torch.bfloat16, seed=1), rand(40, 96, dtype=torch.bfloat16, seed=2)
    clean = mlp_ops.linear_act(x, w, act="gelu")
    bad = x.clone()
    bad[3, 5], bad[64, 0] = float("nan"), float("inf")
    y = mlp_ops.linear_act(bad, w, act="gelu")
    hit = torch.zeros(70, dtype=torch.bool, device="cuda")
    hit[[3, 64]] = True
    assert torch.equal(y[~hit], clean[~hit]) and torch.isnan(y[3]).all() and not torch.isfinite(y[64]).any() | (y[64] == 0).all()
    n, nb = mlp_ops.rms_norm_rows(x), mlp_ops.rms_norm_rows(bad)
    assert torch.equal(n[~hit], nb[~hit]) and torch.isnan(nb[3]).all()
    assert (mlp_ops.rms_norm_rows(torch.zeros(2, 64, device="cuda")) == 0).all()


# ---- together -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 77])
def test_res_mlp(dtype, rows):
    """Norm, product, product as one block, forward, backward and in 8 bits, against 64 bits with a norm-wise tolerance:
    the roundings on the way (y, u, dz, du: half a step each, of values that are averaged) and those of the result."""
    torch.manual_seed(0)
    m = blocks.ResMLP(64, 160, act="silu").to("cuda", dtype)
    x, r = rand(rows, 64, dtype=dtype, seed=1).requires_grad_(), rand(rows, 64, dtype=dtype, seed=2)
    out = m(x, residual=r)
    params = [m.norm.weight, m.lin1.weight, m.lin1.bias, m.lin2.weight, m.lin2.bias]
    g = rand(rows, 64, dtype=dtype, seed=3)
    grads = torch.autograd.grad(out, [x] + params, g)
    p64 = [t.detach().double().requires_grad_() for t in [x] + params]
    h = p64[0] + r.double()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + m.norm.eps) * p64[1]
    u = y @ p64[2].t() + p64[3]
    out64 = (u * torch.sigmoid(u)) @ p64[4].t() + p64[5] + h
    g64 = torch.autograd.grad(out64, p64, g.double())
    tol = 12 * half_step(dtype) + 1e-6
    for a, b in zip((out, *grads), (out64, *g64)):
        assert ((a.double() - b).norm() / b.norm()).item() <= tol
    m8 = m.e4m3()
    out8 = m8(x.detach(), residual=r)
    # two 8-bit products of two operands each, every value off by at most 2^-4: norm-wise under 4 * 2^-4 of the branch
    branch = (out64 - h).detach()
    assert ((out8.double() - out64).norm() / branch.norm()).item() <= 4 * 2.0 ** -4 + tol * (out64.norm() / branch.norm()).item()
    assert sorted(m8.state_dict()) == ["bias1", "bias2", "norm_weight", "scale1", "scale2", "weight1", "weight2"]


def test_graph_replays():
    """Forward, backward and the 8-bit block captured and replayed on changing inputs, with eager work between."""
    torch.manual_seed(0)
    m = blocks.ResMLP(96, 256, act="gelu").to("cuda", torch.bfloat16)
    m8 = m.e4m3()
    x = rand(200, 96, dtype=torch.bfloat16, seed=1).requires_grad_()
    g = rand(200, 96, dtype=torch.bfloat16, seed=2)
    leaves = [x] + list(m.parameters())

    def step():
        out = m(x)
        return [out.detach(), *torch.autograd.grad(out, leaves, g), m8(x.detach())]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(rand(200, 96, dtype=torch.bfloat16, seed=10 + k))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, step()):
            assert torch.equal(a, b)


def test_other_stream_and_repeatability():
    x, w = rand(300, 256, dtype=torch.bfloat16, seed=1), rand(512, 256, dtype=torch.bfloat16, seed=2, scale=0.06)
    want = mlp_ops.linear_act(x, w, act="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        runs = [mlp_ops.linear_act(x, w, act="gelu") for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(r, want) for r in runs)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_second_derivative(dtype):
    """create_graph gives the same gradients; what differentiates them again raises instead of seeing constants."""
    x, w = rand(7, 40, dtype=dtype, seed=1).requires_grad_(), rand(24, 40, dtype=dtype, seed=2).requires_grad_()
    b, r = rand(24, dtype=dtype, seed=3).requires_grad_(), rand(7, 24, dtype=dtype, seed=4).requires_grad_()
    n, s = rand(40, dtype=dtype, seed=5).requires_grad_(), rand(7, 40, dtype=dtype, seed=6).requires_grad_()
    for out, leaves in ((mlp_ops.linear_act(x, w, b, "silu", r), (x, w, b, r)), (mlp_ops.rms_norm_rows(x, n, 1e-6, s)[0], (x, n, s))):
        first = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
        again = torch.autograd.grad(out, leaves, torch.ones_like(out), create_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
        with pytest.raises(RuntimeError, match="no second derivative"):
            again[0].float().square().sum().backward()


def test_only_some_inputs_need_gradients():
    """Each subset of the inputs that asks for a gradient gets the one that it gets among all."""
    dtype = torch.bfloat16
    make = [lambda: rand(33, 64, dtype=dtype, seed=1), lambda: rand(48, 64, dtype=dtype, seed=2, scale=0.2),
            lambda: rand(48, dtype=torch.float32, seed=3), lambda: rand(33, 48, dtype=dtype, seed=4)]
    norm = [lambda: rand(33, 64, dtype=dtype, seed=1), lambda: rand(64, dtype=torch.float32, seed=2),
            lambda: rand(33, 64, dtype=dtype, seed=3)]

    def linear(t):
        return mlp_ops.linear_act(t[0], t[1], t[2], "gelu", t[3])

    def rms(t):
        y, h = mlp_ops.rms_norm_rows(t[0], t[1], 1e-6, t[2])
        return y + h
    for inputs, op in ((make, linear), (norm, rms)):
        for absent in (None, 2, 3)[:len(inputs) - 1]:
            want = None
            for mask in reversed(range(1, 1 << len(inputs))):
                t = [f() for f in inputs]
                if absent is not None and op is linear:
                    if mask >> absent & 1:
                        continue
                    t[absent] = None
                for k, v in enumerate(t):
                    if mask >> k & 1:
                        v.requires_grad_()
                out = op(t)
                out.backward(rand(*out.shape, dtype=dtype, seed=9))
                got = {k: v.grad for k, v in enumerate(t) if v is not None}
                want = want or got
                for k, v in got.items():
                    assert torch.equal(v, want[k]) if mask >> k & 1 else v is None


def test_calls_from_threads_on_their_own_streams():
    """Calls at once share no memory: each thread's forward and backward on its own stream gives what it gives alone."""
    import threading
    dtype = torch.bfloat16
    w = rand(520, 264, dtype=dtype, seed=2, scale=0.1)
    xs = [rand(300 + 8 * k, 264, dtype=dtype, seed=10 + k) for k in range(4)]

    def step(x):
        a, v = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = mlp_ops.linear_act(mlp_ops.rms_norm_rows(a), v, act="gelu")
        return [y.detach(), *torch.autograd.grad(y, (a, v), torch.ones_like(y))]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    got = [None] * len(xs)

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(8):
                got[k] = step(xs[k])
            stream.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert a is not None and all(torch.equal(p, q) for p, q in zip(a, b))


def test_offsets_beyond_32_bits():
    """2.3e9 elements a tensor: a thousand rows repeated give the thousand's results in the first and in the last block, bit for
    bit (rows do not see each other; the products' operands are -1, 0 and 1, so that every sum is exact in any order)."""
    n, C, blocks_, dtype = 1000, 16384, 140, torch.bfloat16

    def whole(t):
        return t.repeat(blocks_, *([1] * (t.dim() - 1)))

    def same(big, small):
        parts = big.view(blocks_, n, *big.shape[1:])
        return torch.equal(parts[0], small) and torch.equal(parts[-1], small)
    base, g = rand(n, C, dtype=dtype, seed=1), rand(n, C, dtype=dtype, seed=2)
    weight = rand(C, dtype=dtype, seed=3)
    big, big_g = whole(base), whole(g)
    out = []
    for x, up in ((base, g), (big, big_g)):
        leaf = x.detach().requires_grad_()
        y, h = mlp_ops.rms_norm_rows(leaf, weight, 1e-6, x)
        dx, = torch.autograd.grad(y, (leaf,), up)
        out.append((y.detach(), h.detach(), dx, *mlp_ops.quantize_rows(x)))
        del leaf, y, h, dx
    for k, (small, large) in enumerate(zip(*out)):
        assert same(large.view(torch.uint8) if k == 3 else large, small.view(torch.uint8) if k == 3 else small), k
    del out, big, big_g

    gen = torch.Generator().manual_seed(4)

    def signs(*shape):
        return torch.randint(-1, 2, shape, generator=gen).to(dtype).cuda()
    x, w, up = signs(n, C), signs(64, C), signs(n, 64)               # long rows in: x and dx are large
    bx = whole(x).requires_grad_()
    bw = w.detach().requires_grad_()
    y = mlp_ops.linear_act(bx, bw)
    dx, dw = torch.autograd.grad(y, (bx, bw), whole(up))
    assert same(y.detach(), (x.float() @ w.float().t()).to(dtype)) and same(dx, (up.float() @ w.float()).to(dtype))
    assert torch.equal(dw, ((up.float().t() @ x.float()) * blocks_).to(dtype))
    del bx, y, dx
    x, w, r, up = signs(n, 64), signs(C, 64), signs(n, C), signs(n, C)   # long rows out: y, what is kept and g are large
    bx, bw = whole(x).requires_grad_(), w.detach().requires_grad_()
    y = mlp_ops.linear_act(bx, bw, act="relu", residual=whole(r))
    dx, dw = torch.autograd.grad(y, (bx, bw), whole(up))
    z = x.float() @ w.float().t()
    assert same(y.detach(), (z.clamp_min(0) + r.float()).to(dtype))
    dz = up.float() * (z > 0)
    assert same(dx, (dz @ w.float()).to(dtype)) and torch.equal(dw, ((dz.t() @ x.float()) * blocks_).to(dtype))


def test_norm_layer_and_pre_activation():
    from deep_gcns_torch_amd import node_ops
    from deep_gcns_torch_amd.gcn_lib.sparse.torch_nn import MLP, norm_layer
    x = rand(500, 64, dtype=torch.float32, seed=1)
    norm = norm_layer("rms", 64).cuda()
    y, skip = node_ops.pre_activation(norm, x, skip=True)
    h64, _, y64 = norm_ref(x, norm.weight, None, norm.eps)
    within(y, y64.clamp_min(0), y_bound(y64, 64, torch.float32))
    assert skip is x
    mlp = MLP([64, 128, 32], norm="rms", last_lin=True).cuda()
    assert mlp(x).shape == (500, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, C", [(300, 128), (64, 1001), (40, 4096), (16, 16384), (3, 32768)])
def test_rows_e4m3_are_divided(dtype, rows, C):
    """The bits of the same thing in torch, ties included: scale = max|x| / 448, q = x / scale (both rounded to fp32, q then to e4m3)."""
    x = rand(rows, C, dtype=dtype, seed=1, scale=3.0).float()
    x[0] *= 1e-36 if dtype != torch.float16 else 1.0                # a scale among the least normal numbers
    x = x.to(dtype)
    q = mlp_ops.quantize_rows(x)
    scale = x.float().abs().amax(-1) / 448.0
    assert torch.equal(q.scale, scale.clamp_min(torch.finfo(torch.float32).tiny))
    want = (x.float() / q.scale.unsqueeze(-1)).to(torch.float8_e4m3fn)
    assert torch.equal(q.data.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, C", [(1, 4096), (130, 513), (257, 33), (2000, 128), (17, 8191), (2, 32768)])
def test_norm_gradients_see_the_sum(dtype, rows, C):
    """The gradients with a residual are those of the fp32 sum x + r, not of h as it is stored: an fp32 weight's gradient
    shows it, which has no rounding of its own.  Terms g xh with a sum of `rows` and one of C fp32 roundings."""
    x, r = rand(rows, C, dtype=dtype, seed=1).requires_grad_(), rand(rows, C, dtype=dtype, seed=2).requires_grad_()
    w = (1 + rand(C, dtype=torch.float32, seed=3, scale=0.3)).requires_grad_()
    g, gh = rand(rows, C, dtype=dtype, seed=4), rand(rows, C, dtype=dtype, seed=5)
    y, h = mlp_ops.rms_norm_rows(x, w, eps=1e-5, residual=r)
    gx, gw, gr = torch.autograd.grad((y, h), (x, w, r), (g, gh))
    h64, rstd, _ = norm_ref(x.detach(), w.detach(), r.detach(), 1e-5)
    xh, g64, rel = h64 * rstd, g.double(), (C + 20) * U
    gw64 = (g64 * xh).sum(0)
    within(gw, gw64, (g64 * xh).abs().sum(0) * (rows + C + 20) * U + gw64.abs() * U + TINY[torch.float32], "gw")
    gg = g64 * w.detach().double()
    dot = (gg * xh).mean(-1, keepdim=True)
    dx = rstd * (gg - xh * dot) + gh.double()
    edx = rstd * (xh.abs() * (gg * xh).abs().mean(-1, keepdim=True) * rel + (xh * dot).abs() * rel + gg.abs() * rel)
    edx = edx + rstd * (gg.abs() + (xh * dot).abs()) * 8 * U + gh.double().abs() * 2 * U
    within(gx, dx, edx + dx.abs() * (half_step(dtype) * 1.01 + 2 * U) + TINY[dtype], "gx")
    assert torch.equal(gx, gr)
    one, wide = r.detach()[:1].expand(rows, C), torch.cat([x.detach(), x.detach()], 1)[:, :C]      # strides that the backward meets again
    for a, b in ((wide, one), (one, wide)):
        got, want = ([t.requires_grad_() for t in pair] for pair in ((a.detach(), b.detach()), (a.clone(), b.clone())))
        both = [torch.autograd.grad(mlp_ops.rms_norm_rows(p, w, 1e-5, q)[0], (p, w, q), g) for p, q in (got, want)]
        assert all(torch.equal(s, t) for s, t in zip(*both))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act, low, high", [("gelu", -7.0, -2.0), ("silu", -28.0, -3.0)])
@pytest.mark.parametrize("rows", [9, 700])
def test_gradients_of_saturated_units(dtype, act, low, high, rows):
    """One product per result, so that z is x to the bit: dx = act'(z) g within, relative to it, the kept slope's half step of
    2^-10, dz's and dx's roundings (the second of a value that has them already), and 2^-12 for the slope's own evaluation
    (the distribution function's fit 1e-5, its difference from z times the density at most doubled from z = -2 on, the
    exponential's argument z^2 / 2 2^-24)."""
    x = torch.linspace(low, high, rows, device="cuda").to(dtype).view(rows, 1).requires_grad_()
    w = torch.ones(1, 1, device="cuda", dtype=dtype)
    g = torch.full((rows, 1), 1024.0, device="cuda", dtype=dtype)
    gx, = torch.autograd.grad(mlp_ops.linear_act(x, w, act=act), x, g)
    want = act_ref(x.detach().double(), act)[1] * 1024
    within(gx, want, want.abs() * (half_step(dtype) + 2.0 ** -10 + 2.0 ** -12) + TINY[dtype], act)
    assert (gx < 0)[want < -TINY[dtype]].all()                       # (what fp16 itself rounds to 0: 1024 slope under 2^-25)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("rows, N", [(1, 40), (4, 64), (16, 8200), (16, 4096)])
def test_few_e4m3_rows_are_summed_in_fp32(out, rows, N):
    """2^16 - 2^16 + 2^(16 - d): up to 16 rows nothing is cut from a product, whatever the result's type."""
    for where, d in ((2, 13), (2, 14), (7, 18), (8, 20), (40, 26)):
        x, w = torch.zeros(rows, 160, device="cuda"), torch.zeros(N, 160, device="cuda")
        x[:, 0], w[:, 0], x[:, 1], w[:, 1] = 256.0, 256.0, 256.0, -256.0
        x[:, where], w[:, where] = 2.0 ** ((17 - d) // 2), 2.0 ** (16 - d - (17 - d) // 2)
        rows8 = [RowsE4M3(t.to(torch.float8_e4m3fn), torch.ones(t.size(0), device="cuda")) for t in (x, w)]
        y = mlp_ops.linear_act_e4m3(*rows8, out_dtype=out)
        assert torch.equal(y.float(), torch.full((rows, N), 2.0 ** (16 - d), device="cuda")), (where, d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, K, N", [(1, 1, 1), (3, 64, 40), (16, 1030, 70), (70, 96, 40), (300, 130, 264), (130, 6152, 136), (40, 33, 4100)])
def test_infinite_operands_of_products(dtype, rows, K, N):
    """Infinities, NaN and zeros against them give what the products of the definition give, in the forward and in both
    products of the backward; everything else keeps its bounds."""
    x, w, g = (rand(*s, dtype=dtype, seed=k, scale=c) for k, (s, c) in enumerate((((rows, K), 1.0), ((N, K), K ** -0.5), ((rows, N), 1.0))))
    inf, nan = float("inf"), float("nan")
    x[0, K // 2] = inf
    w[N // 2, K // 2] = 0.0                                          # against the infinity: NaN
    if rows > 2:
        x[rows - 1, K - 1], x[1, 0] = -inf, nan
        w[N - 1, 0] = -inf
        g[rows // 2, N // 3] = inf
        x[rows // 2, K // 3] = 0.0

    def like(got, want, bound, what):
        got, finite = got.double(), torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), what
        assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf()), what
        assert ((got - want).abs()[finite] <= bound[finite]).all(), what

    def product(a, b):                                               # (..., k) x (n, k), and the sum of its finite terms' magnitudes
        a, b = a.double().cpu(), b.double().cpu()
        return (a @ b.t()).cuda(), (a.abs().nan_to_num(0, 0, 0) @ b.abs().nan_to_num(0, 0, 0).t()).cuda()

    def bounds(z, mag, k):
        return mag * (6 * k + 12) * U + z.abs() * half_step(dtype) * 1.01 + TINY[dtype]
    z, mag = product(x, w)
    like(mlp_ops.linear_act(x, w), z, bounds(z, mag, K), "z")
    y = torch.where(z < 0, torch.zeros_like(z), z)                   # relu keeps NaN, and takes -inf to 0
    like(mlp_ops.linear_act(x, w, act="relu"), y, bounds(z.nan_to_num(0, 0, 0), mag, K), "relu")
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(mlp_ops.linear_act(a, b), (a, b), g)
    for got, (want, mag), k, what in ((dx, product(g, w.t()), N, "dx"), (dw, product(g.t(), x.t()), rows, "dw")):
        like(got, want, bounds(want, mag, k), what)


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_raises(grad_mode):
    """A tangent is never dropped: neither operator has a forward-mode derivative, and each says so."""
    import torch.autograd.forward_ad as fw
    x, w = rand(40, 64, dtype=torch.float32, seed=1), rand(64, 64, dtype=torch.float32, seed=2)
    b, q = rand(64, dtype=torch.float32, seed=3), mlp_ops.quantize_rows(rand(40, 64, dtype=torch.float32, seed=4))
    with torch.set_grad_enabled(grad_mode), fw.dual_level():
        d, dw, db = fw.make_dual(x, x), fw.make_dual(w, w), fw.make_dual(b, b)
        ds = RowsE4M3(q.data, fw.make_dual(q.scale, q.scale))
        q40 = RowsE4M3(q.data, q.scale)
        for call in (lambda: mlp_ops.linear_act(d, w), lambda: mlp_ops.linear_act(x, dw), lambda: mlp_ops.linear_act(x, w, db),
                     lambda: mlp_ops.linear_act(x, w, residual=d), lambda: mlp_ops.rms_norm_rows(d), lambda: mlp_ops.rms_norm_rows(x, db),
                     lambda: mlp_ops.rms_norm_rows(x, b, residual=d), lambda: mlp_ops.rms_norm_rows_e4m3(d, b),
                     lambda: mlp_ops.quantize_rows(d), lambda: mlp_ops.linear_act_e4m3(ds, q40, out_dtype=torch.float32),
                     lambda: mlp_ops.linear_act_e4m3(q40, ds, out_dtype=torch.float32)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
    with fw.dual_level():                                            # a tangent of the gradient that a backward is given
        for out, leaf in (((lambda t: mlp_ops.linear_act(t, w)), x), (mlp_ops.rms_norm_rows, x)):
            leaf = leaf.clone().requires_grad_()
            y = out(leaf)
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(y, leaf, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))
    for op in (lambda t: mlp_ops.linear_act(t, w), mlp_ops.rms_norm_rows, lambda t: mlp_ops.quantize_rows(t).scale):
        with pytest.raises(RuntimeError):
            torch.func.jvp(op, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.vmap(op)(x)


def test_e4m3_values_that_want_a_gradient_raise():
    x = rand(20, 64, dtype=torch.float32, seed=1)
    one = torch.ones(20, device="cuda")
    plain, wants = RowsE4M3(x.to(torch.float8_e4m3fn), one), RowsE4M3(x.clone().requires_grad_().to(torch.float8_e4m3fn), one)
    assert wants.data.requires_grad
    for args in ((wants, plain), (plain, wants)):
        with pytest.raises(RuntimeError, match="has no gradient"):
            mlp_ops.linear_act_e4m3(*args)
        with torch.no_grad():
            assert torch.equal(mlp_ops.linear_act_e4m3(*args), mlp_ops.linear_act_e4m3(plain, plain))


def test_work_is_on_the_current_stream():
    """Inputs that the side stream writes behind a long product: work on any other stream would read what was there before."""
    dtype = torch.bfloat16
    first, second = rand(300, 256, dtype=dtype, seed=1), rand(300, 256, dtype=dtype, seed=2)
    w, n = rand(512, 256, dtype=dtype, seed=3, scale=0.06), rand(256, dtype=dtype, seed=4)
    w8 = mlp_ops.quantize_rows(w)

    def step(x):
        leaf, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = mlp_ops.linear_act(mlp_ops.rms_norm_rows(leaf, n), wl, act="gelu")
        grads = torch.autograd.grad(y, (leaf, wl), torch.ones_like(y))
        with torch.no_grad():
            q = mlp_ops.quantize_rows(x)
            return [y.detach(), *grads, q.data.view(torch.uint8), q.scale, mlp_ops.linear_act_e4m3(q, w8),
                    mlp_ops.rms_norm_rows_e4m3(x, n)[0].view(torch.uint8)]
    want, old = step(second), step(first)
    x, big = first.clone(), torch.randn(8192, 8192, device="cuda")
    out = torch.empty_like(big)
    torch.mm(big, big, out=out)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(4):
            torch.mm(big, big, out=out)
        x.copy_(second)
        got = step(x)
        assert not side.query()                                      # all of it was queued while the product ran
    side.synchronize()
    for a, b, c in zip(got, want, old):
        assert torch.equal(a, b) and not torch.equal(a, c)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_backward_entry_of_a_stored_sum(dtype):
    """dgcn_rms_norm_bwd takes h itself: without a residual the same bits as the operator's backward."""
    from deep_gcns_torch_amd import _lib
    lib, rows, C = _lib.load(), 70, 513
    h, g = rand(rows, C, dtype=dtype, seed=1), rand(rows, C, dtype=dtype, seed=2)
    w = (1 + rand(C, dtype=torch.float32, seed=3, scale=0.3)).requires_grad_()
    leaf = h.clone().requires_grad_()
    want = torch.autograd.grad(mlp_ops.rms_norm_rows(leaf, w), (leaf, w), g)
    code, y, rstd = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], torch.empty_like(h), torch.empty(rows, device="cuda")
    dx, dw = torch.empty_like(h), torch.empty(C, device="cuda")
    parts = torch.empty(lib.dgcn_rms_norm_num_partials(rows, C), C, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.dgcn_rms_norm_fwd(h.data_ptr(), C, None, 0, w.data_ptr(), 1, 1e-6, code, y.data_ptr(), None, None, None, rstd.data_ptr(),
                                 rows, C, stream) == 0
    assert lib.dgcn_rms_norm_bwd(g.data_ptr(), C, None, 0, h.data_ptr(), C, w.data_ptr(), 1, rstd.data_ptr(), code, dx.data_ptr(),
                                 dw.data_ptr(), parts.data_ptr(), rows, C, stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
