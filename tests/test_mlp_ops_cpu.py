"""mlp_ops without a GPU: refusals of the entry points, and argument errors of the C entry points (nothing is launched)."""
import ctypes as C

import pytest
import torch

from deep_gcns_torch_amd import _lib, blocks, mlp_ops
from deep_gcns_torch_amd.mlp_ops import RowsE4M3

X, W = torch.randn(3, 8), torch.randn(5, 8)


def _e4m3(rows, k):
    return RowsE4M3(torch.randn(rows, k).to(torch.float8_e4m3fn), torch.ones(rows))


@pytest.mark.parametrize("call, error, text", [
    (lambda: mlp_ops.rms_norm_rows(X.double()), TypeError, "float32, bfloat16 or float16"),
    (lambda: mlp_ops.rms_norm_rows(torch.zeros(())), ValueError, "last dimension"),
    (lambda: mlp_ops.rms_norm_rows(torch.zeros(3, 0)), ValueError, "last dimension"),
    (lambda: mlp_ops.rms_norm_rows(torch.zeros(1, 32769)), ValueError, "at most 32768"),
    (lambda: mlp_ops.rms_norm_rows(X, torch.ones(7)), ValueError, r"weight must have shape \(8,\)"),
    (lambda: mlp_ops.rms_norm_rows(X, torch.ones(8, dtype=torch.float16)), TypeError, "weight must be"),
    (lambda: mlp_ops.rms_norm_rows(X, residual=X[:2]), ValueError, "residual must have shape"),
    (lambda: mlp_ops.rms_norm_rows(X, residual=X.half()), TypeError, "residual must be"),
    (lambda: mlp_ops.rms_norm_rows(X), RuntimeError, "no CPU fallback"),
    (lambda: mlp_ops.rms_norm_rows_e4m3(X), RuntimeError, "no CPU fallback"),
    (lambda: mlp_ops.quantize_rows(torch.zeros(1, 32769)), ValueError, "at most 32768"),
    (lambda: mlp_ops.quantize_rows(X.long()), TypeError, "float32, bfloat16 or float16"),
    (lambda: mlp_ops.quantize_rows(X), RuntimeError, "no CPU fallback"),
    (lambda: mlp_ops.linear_act(X, W.half()), TypeError, "weight must be"),
    (lambda: mlp_ops.linear_act(X, W[:, :7]), ValueError, "weight"),
    (lambda: mlp_ops.linear_act(X, W[0]), ValueError, "weight"),
    (lambda: mlp_ops.linear_act(X, W[:0]), ValueError, "N >= 1"),
    (lambda: mlp_ops.linear_act(X, torch.zeros(1, 8).expand((1 << 20) + 1, 8)), ValueError, "at most"),
    (lambda: mlp_ops.linear_act(X, W, torch.ones(4)), ValueError, r"bias must have shape \(5,\)"),
    (lambda: mlp_ops.linear_act(X, W, torch.ones(5).half()), TypeError, "bias must be"),
    (lambda: mlp_ops.linear_act(X, W, act="tanh"), ValueError, "act must be one of"),
    (lambda: mlp_ops.linear_act(X, W, residual=torch.ones(5)), ValueError, "residual must have shape"),
    (lambda: mlp_ops.linear_act(X, W, residual=torch.ones(3, 5).half()), TypeError, "residual must be"),
    (lambda: mlp_ops.linear_act(X, W), RuntimeError, "no CPU fallback"),
    (lambda: mlp_ops.linear_act_e4m3(RowsE4M3(X, torch.ones(3)), _e4m3(5, 8)), TypeError, "float8_e4m3fn"),
    (lambda: mlp_ops.linear_act_e4m3(_e4m3(3, 8), RowsE4M3(_e4m3(5, 8).data, torch.ones(4))), ValueError, "scales of shape"),
    (lambda: mlp_ops.linear_act_e4m3(_e4m3(3, 8), _e4m3(5, 8), out_dtype=torch.float64), TypeError, "out_dtype"),
    (lambda: mlp_ops.linear_act_e4m3(_e4m3(3, 8), _e4m3(5, 8), residual=torch.ones(3, 5)), TypeError, "residual must be"),
    (lambda: mlp_ops.linear_act_e4m3(_e4m3(3, 8), _e4m3(5, 8)), RuntimeError, "no CPU fallback"),
    (lambda: blocks.ResMLP(8, 16, act="tanh"), ValueError, "act must be one of"),
])
def test_refusals(call, error, text):
    with pytest.raises(error, match=text):
        call()


def test_c_entry_argument_errors_do_not_launch():
    lib = _lib.load()
    buf = (C.c_float * 64)()
    p = (C.addressof(buf) + 15) & ~15
    norm = lib.dgcn_rms_norm_fwd
    assert norm(None, 8, None, 0, None, 0, 1e-6, 0, p, None, None, None, None, 1, 8, None) == -1
    assert norm(p, 8, None, 0, None, 0, 1e-6, 0, p, None, p, p, None, 1, 8, None) == -4        # y and q
    assert norm(p, 8, None, 0, None, 0, 1e-6, 0, None, None, p, None, None, 1, 8, None) == -1  # q without scales
    assert norm(p, 8, None, 0, None, 0, 1e-6, 3, p, None, None, None, None, 1, 8, None) == -4  # 8-bit rows have no norm
    assert norm(p, 8, None, 0, None, 0, 1e-6, 0, p, None, None, None, None, 1, 32769, None) == -2
    assert norm(p, 8, None, 0, None, 0, 1e-6, 0, p, None, None, None, None, 0, 8, None) == 0   # no rows: no launch
    bwd = lib.dgcn_rms_norm_bwd
    assert bwd(p, 8, None, 0, p, 8, None, 0, p, 0, None, None, None, 1, 8, None) == -1          # nothing asked for
    assert bwd(p, 8, None, 0, p, 8, None, 0, p, 0, p, p, None, 1, 8, None) == -1                # dw without its partials
    assert bwd(p, 8, None, 0, p, 8, None, 0, p, 0, p, None, None, 0, 8, None) == -2             # a sum over no rows is the caller's
    assert lib.dgcn_quantize_rows_e4m3(p, 8, 0, p, None, 1, 8, None) == -1
    assert lib.dgcn_param_sum(None, 1, 4, 0, p, None) == -1
    assert lib.dgcn_rms_norm_num_partials(0, 8) == 0
    act = lib.dgcn_linear_act
    assert act(p, 8, p, 8, None, None, None, 0, None, 0, 0, 0.0, 3, 1, None, p, 1, 8, 8, None, 0, None) == -1   # e4m3 without scales
    assert act(p, 8, p, 8, None, None, None, 0, None, 0, 0, 0.0, 1, 2, None, p, 1, 8, 8, None, 0, None) == -4   # bf16 rows, fp16 result
    assert act(p, 8, p, 8, None, None, None, 0, None, 0, 9, 0.0, 1, 1, None, p, 1, 8, 8, None, 0, None) == -4   # no such activation
    assert act(p, 8, p, 8, None, None, None, 0, None, 0, 0, 0.0, 1, 1, None, p, 1, 8, 8, p + 4, 0, None) == -3  # workspace alignment
    assert act(p, 8, p, 8, None, None, None, 0, None, 0, 0, 0.0, 1, 1, None, p, 1, 0, 8, None, 0, None) == -2
    back = lib.dgcn_linear_bwd
    assert back(p, 8, p, 8, p, 8, None, 1, 0.0, 0, p, p, p, 0, 1, 8, 8, None, 0, None) == -1                    # an activation needs z
    assert back(p, 8, p, 8, p, 8, p, 9, 0.0, 0, p, p, p, 0, 1, 8, 8, None, 0, None) == -4
    assert back(p, 8, p, 8, p, 8, None, 0, 0.0, 0, p, p, p, 0, 0, 8, 8, None, 0, None) == -2
    assert back(p, 8, p, 8, p, 8, None, 0, 0.0, 0, None, None, None, 0, 1, 8, 8, None, 0, None) == 0            # nothing asked for
    # workspaces: none for few rows; partial sums for a long reduction; copies for rows off dwords, and too small is refused
    need, back_need = lib.dgcn_linear_workspace, lib.dgcn_linear_bwd_workspace
    assert need(p, 8, p, 8, 1, 16, 8, 8) == 0 and need(p, 4096, p, 4096, 1, 65536, 4096, 4096) == 0
    assert need(p, 10, p, 8, 1, 1000, 8, 8) == 0 and need(p, 9, p, 8, 1, 1000, 8, 8) >= 1000 * 16 and need(p + 2, 8, p, 8, 1, 1000, 8, 8) >= 1000 * 16
    assert act(p + 2, 8, p, 8, None, None, None, 0, None, 0, 0, 0.0, 1, 1, None, p, 1000, 8, 8, p, 64, None) == -5
    n = back_need(p, 64, p, 64, p, 64, 0, 1, 2, 100000, 64, 64)
    assert n > 0 and back(p, 64, p, 64, p, 64, None, 0, 0.0, 1, None, p, None, 0, 100000, 64, 64, p, n - 256, None) == -5


def test_norm_layer_offers_rms():
    from deep_gcns_torch_amd.gcn_lib.sparse.torch_nn import norm_layer
    m = norm_layer("rms", 12)
    assert isinstance(m, mlp_ops.RMSNorm) and list(m.state_dict()) == ["weight"] and m.weight.shape == (12,)


def test_missing_host_extension_raises(monkeypatch):
    import sys
    import deep_gcns_torch_amd
    monkeypatch.setattr(mlp_ops, "_host", None)
    monkeypatch.delattr(deep_gcns_torch_amd, "_mlp_host", raising=False)
    monkeypatch.setitem(sys.modules, "deep_gcns_torch_amd._mlp_host", None)
    with pytest.raises(RuntimeError, match="python -m deep_gcns_torch_amd.build"):
        mlp_ops.quantize_rows(torch.zeros(2, 8))


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.float(), lambda m: torch.nn.Sequential(m).bfloat16()[0],
                                  lambda m: m.to("cpu", torch.float16), lambda m: m.to("meta")])
def test_casts_leave_e4m3_weights(cast, monkeypatch):
    """A module's cast converts its parameters in 16 and 32 bits, and neither the 8-bit weights nor their scales."""
    def plain(x):
        scale = x.abs().amax(-1) / 448
        return RowsE4M3((x / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), scale)
    monkeypatch.setattr(mlp_ops, "quantize_rows", plain)
    m = blocks.ResMLP(24, 40).e4m3()
    before, names = {k: v.clone() for k, v in m.state_dict().items()}, list(m.state_dict())
    got = cast(m)
    assert list(got.state_dict()) == names
    for k in ("weight1", "scale1", "weight2", "scale2"):
        t = got.state_dict()[k]
        assert t.dtype == before[k].dtype and t.shape == before[k].shape
        if t.device.type == "cpu":
            view = torch.uint8 if "weight" in k else torch.int32
            assert torch.equal(t.view(view), before[k].view(view))
    assert len({got.state_dict()[k].device for k in names}) == 1
    assert len({got.state_dict()[k].dtype for k in ("norm_weight", "bias1", "bias2")}) == 1


def test_norm_of_a_sum_backward_argument_errors_do_not_launch():
    lib = _lib.load()
    buf = (C.c_float * 64)()
    p = (C.addressof(buf) + 15) & ~15
    bwd = lib.dgcn_rms_norm_sum_bwd
    ok = dict(g=p, ldg=8, gh=None, ldgh=0, x=p, ldx=8, res=p, ldr=8, w=None, w_f32=0, rstd=p, dtype=0, dx=p, dw=None, parts=None,
              rows=1, C=8, stream=None)

    def rc(**change):
        return bwd(*{**ok, **change}.values())
    for change in (dict(g=None), dict(x=None), dict(rstd=None), dict(dx=None), dict(dw=p)):
        assert rc(**change) == -1, change                                     # (dw without its partials)
    for change in (dict(rows=0), dict(C=0), dict(C=32769), dict(ldx=-1), dict(ldr=-1), dict(ldg=-1), dict(gh=p, ldgh=-1)):
        assert rc(**change) == -2, change
    assert rc(dtype=3) == -4
