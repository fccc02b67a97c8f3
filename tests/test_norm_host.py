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


def test_checkpoints_of_group_norm_models_name_their_groups(tmp_path):
    """The group count is no part of a state_dict: it is recorded, given, or refused."""
    import ugpg
    state = ugpg.PGUNet1(3, 1, norm="group", groups=8).state_dict()
    bare, full = tmp_path / "bare.pth", tmp_path / "full.pth"
    torch.save({"model_state_dict": state, "stage": 1}, bare)
    torch.save({"model_state_dict": state, "stage": 1, "norm_groups": 8}, full)
    for path, groups in ((full, None), (full, 8), (bare, 8)):
        t = ugpg.MoNuSegTester(str(path), device="cpu", norm_groups=groups)
        assert t.model.inc.conv.conv_op[1].num_groups == 8
    for path, groups in ((bare, None), (full, 16)):
        with pytest.raises(RuntimeError, match="norm_groups"):
            ugpg.MoNuSegTester(str(path), device="cpu", norm_groups=groups)
    tr = ugpg.UncertaintyGuidedProgressiveTrainer(3, 1, device="cpu", norm="group", norm_groups=16)
    with pytest.raises(ValueError, match="8 norm groups"):
        tr.load_stage_weights(1, str(full))


def test_one_logit_cannot_be_distilled():
    from ugpg.herlev import HerlevTrainer
    with pytest.raises(ValueError, match="at least 2 classes"):
        HerlevTrainer({"num_classes": 1, "epochs_per_stage": 1, "distill_weight": 0.5, "device": "cpu"})


def test_c_entries_refuse_before_any_launch():
    import ctypes as C
    from ugpg import _C
    lib, p = _C.lib, 0x1000  # never dereferenced on the host

    def desc(**kw):
        f = dict(x=p, dtype=0, B=2, HW=64, C=32, G=4, gamma=None, beta=None, eps=1e-5, act=1, mean=p, rstd=p)
        f.update(kw)
        return C.byref(_C.GroupNormDesc(*f.values()))
    sizes = (dict(dtype=2), dict(B=0), dict(HW=0), dict(C=30), dict(G=0), dict(G=5), dict(eps=-1.0),
             dict(eps=float("nan")), dict(act=3), dict(act=-1), dict(C=1 << 21, G=1), dict(B=1 << 22, G=8),
             dict(HW=1 << 41))
    big = 1 << 40
    for kw in (*sizes, dict(x=None), dict(x=p + 2), dict(mean=None), dict(rstd=None)):
        assert lib.ugpg_group_norm_fwd(desc(**kw), p, p, big, None) == -1, kw
        assert b"group_norm_fwd" in lib.ugpg_last_error()
        assert lib.ugpg_group_norm_bwd(desc(**kw), p, kw.get("dtype", 0), p, kw.get("dtype", 0), None, None,
                                       None, p, big, None) == -1, kw
        assert b"group_norm_bwd" in lib.ugpg_last_error()
    for kw in sizes:
        assert lib.ugpg_group_norm_workspace(desc(**kw), 0) == 0
        assert lib.ugpg_group_norm_workspace(desc(**kw), 1) == 0
    need, nb = (lib.ugpg_group_norm_workspace(desc(), k) for k in (0, 1))
    assert 0 < need <= nb
    assert lib.ugpg_group_norm_fwd(None, p, p, big, None) == -1
    assert lib.ugpg_group_norm_fwd(desc(), None, p, big, None) == -1
    assert lib.ugpg_group_norm_fwd(desc(), p, p, need - 1, None) == -3
    assert lib.ugpg_group_norm_fwd(desc(), p, None, need, None) == -3
    bwd = lambda d=0, dy=p, dyt=0, dx=p, dxt=0, n=nb: lib.ugpg_group_norm_bwd(
        desc(dtype=d), dy, dyt, dx, dxt, None, None, None, p, n, None)
    assert bwd(n=nb - 1) == -3
    for kw in (dict(dy=None), dict(dx=None), dict(dyt=1), dict(dxt=1), dict(d=1, dyt=1)):
        assert bwd(**kw) == -1, kw


def test_models_take_a_norm():
    """norm="group" keeps the parameter names and drops the running buffers; the default is
    the reference's BatchNorm; anything else, and groups that do not divide, are refused."""
    import torch.nn as nn
    import ugpg
    a, b = ugpg.PGUNet1(3, 1), ugpg.PGUNet1(3, 1, norm="group", groups=16)
    assert [k for k, _ in a.named_parameters()] == [k for k, _ in b.named_parameters()]
    assert isinstance(a.inc.conv.conv_op[1], nn.BatchNorm2d) and not list(b.buffers())
    assert b.inc.conv.conv_op[1].num_groups == 16
    p = ugpg.ProgressiveUNet(3, 1, norm="group")
    assert all(isinstance(p.stages[s].inc.conv.conv_op[1], nn.GroupNorm) for s in p.stages)
    with pytest.raises(ValueError, match="norm must be"):
        ugpg.DoubleConv(3, 64, norm="layer")
    with pytest.raises(ValueError):
        ugpg.DoubleConv(3, 64, norm="group", groups=48)
    state, copied = ugpg.transfer_state(b.state_dict(), ugpg.PGUNet2(3, 1, norm="group", groups=16).state_dict())
    assert len(copied) > 10


def test_autograd_nodes_are_built_from_these_sources():
    import importlib.util
    from pathlib import Path
    from ugpg import _nodes
    root = Path(__file__).resolve().parent.parent
    spec = importlib.util.spec_from_file_location("_b", root / "ug-pg-unet_amd" / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    assert _nodes.nodes().build_id == b.autograd_id()
    with pytest.raises(ImportError, match="stale"):
        _nodes._check_fresh("0" * 32)
