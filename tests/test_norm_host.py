"""Refusals of group_norm_act / GroupNormAct and of their C entries (no GPU needed)."""
import pytest
import torch


def test_group_norm_act_refuses_bad_arguments():
    import ugpg
    x = torch.zeros(2, 3, 3, 12)
    bad = [
        (dict(x=torch.zeros(4), num_groups=1), ValueError, "expected"),
        (dict(x=x, num_groups=5), ValueError, "divide"),
        (dict(x=x, num_groups=0), ValueError, "divide"),
        (dict(x=x, num_groups=2.0), ValueError, "divide"),
        (dict(x=x, num_groups=4, activation="gelu"), ValueError, "activation"),
        (dict(x=x, num_groups=4, eps=-1.0), ValueError, "eps"),
        (dict(x=x, num_groups=4, eps=float("nan")), ValueError, "eps"),
        (dict(x=x.double(), num_groups=4), TypeError, "float32 or bfloat16"),
        (dict(x=x.half(), num_groups=4), TypeError, "float32 or bfloat16"),
        (dict(x=x, num_groups=4, weight=torch.ones(4)), ValueError, "weight"),
        (dict(x=x, num_groups=4, bias=torch.ones(12, dtype=torch.bfloat16)), TypeError, "bias"),
        (dict(x=x, num_groups=4), RuntimeError, "no CPU fallback"),
    ]
    for kw, err, msg in bad:
        with pytest.raises(err, match=msg):
            ugpg.group_norm_act(**kw)


def test_module_refuses_bad_arguments():
    import ugpg
    with pytest.raises(ValueError, match="activation"):
        ugpg.GroupNormAct(4, 12, activation="tanh")
    with pytest.raises(ValueError):
        ugpg.GroupNormAct(5, 12)
    m = ugpg.GroupNormAct(4, 12)
    with pytest.raises(ValueError, match="expected"):
        m(torch.zeros(2, 8, 3, 3))
    assert sorted(m.state_dict()) == ["bias", "weight"]


def test_c_entries_refuse_before_any_launch():
    from ugpg import _C
    lib, p = _C.lib, 0x1000  # never dereferenced on the host
    need = lib.ugpg_group_norm_workspace(2, 64, 32, 4, 0)
    assert need > 0 and lib.ugpg_group_norm_workspace(2, 64, 32, 5, 0) == 0

    def fwd(x=p, dt=0, B=2, hw=64, C=32, G=4, eps=1e-5, act=1, y=p, mean=p, ws=p, n=need):
        return lib.ugpg_group_norm_fwd(x, dt, B, hw, C, G, None, None, eps, act, y, mean, p, ws, n, None)
    for kw in (dict(x=None), dict(dt=2), dict(B=0), dict(hw=0), dict(C=30), dict(G=0), dict(eps=-1.0),
               dict(eps=float("nan")), dict(act=3), dict(act=-1), dict(y=None), dict(mean=None),
               dict(C=1 << 21, G=1), dict(B=1 << 22, G=8), dict(hw=1 << 41)):
        assert fwd(**kw) == -1, kw
        assert b"group_norm_fwd" in lib.ugpg_last_error()
    assert fwd(n=need - 1) == -3 and fwd(ws=None) == -3

    nb = lib.ugpg_group_norm_workspace(2, 64, 32, 4, 1)

    def bwd(dy=p, dyt=0, x=p, dt=0, dx=p, dxt=0, mean=p, G=4, n=nb):
        return lib.ugpg_group_norm_bwd(dy, dyt, x, dt, 2, 64, 32, G, mean, p, None, None, 1, dx, dxt,
                                       None, None, None, p, n, None)
    for kw in (dict(dy=None), dict(x=None), dict(dx=None), dict(mean=None), dict(G=5),
               dict(dyt=1), dict(dxt=1), dict(dt=1, dyt=1), dict(dt=2)):
        assert bwd(**kw) == -1, kw
        assert b"group_norm_bwd" in lib.ugpg_last_error()
    assert bwd(n=nb - 1) == -3
