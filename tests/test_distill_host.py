"""Refusals of teacher_top_logits / distillation_loss and of their C entries (no GPU needed)."""
import ctypes as C

import pytest
import torch


def test_top_logits_refuses_bad_arguments():
    import ugpg
    z = torch.zeros(4, 9)
    for args, err, msg in [((torch.zeros(4), 1), ValueError, "expected"),
                           ((z.half(), 1), TypeError, "float32 or bfloat16"),
                           ((torch.zeros(0, 9), 1), ValueError, "empty"),
                           ((z, 0), ValueError, "k must"), ((z, 10), ValueError, "k must"),
                           ((z, 2.0), ValueError, "k must"), ((torch.zeros(2, 999), 257), ValueError, "k must"),
                           ((z, 3, 0.0), ValueError, "temperature"), ((z, 3, -1.0), ValueError, "temperature"),
                           ((z, 3, float("nan")), ValueError, "temperature"),
                           ((z, 3, 1e-31), ValueError, "temperature"), ((z, 3, 1e31), ValueError, "temperature"),
                           ((z, 3), RuntimeError, "no CPU fallback")]:
        with pytest.raises(err, match=msg):
            ugpg.teacher_top_logits(*args)


def test_distillation_loss_refuses_bad_arguments():
    import ugpg
    z, v, i = torch.zeros(4, 9), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    r, w = torch.zeros(4), torch.ones(4)
    good = dict(logits=z, top=(v, i, r), weight=w)
    for kw, err, msg in [
            (dict(logits=z.double()), TypeError, "float32 or bfloat16"),
            (dict(logits=torch.zeros(5, 9)), ValueError, "do not fit"),
            (dict(top=(torch.zeros(4, 10), torch.zeros(4, 10, dtype=torch.int64), r)), ValueError, "do not fit"),
            (dict(top=(torch.zeros(4, 0), torch.zeros(4, 0, dtype=torch.int64), r)), ValueError, "do not fit"),
            (dict(top=(torch.zeros(4), i, r)), ValueError, "do not fit"),
            (dict(top=(v, i[:, :2], r)), ValueError, "indices"),
            (dict(top=(v, i.to(torch.int16), r)), TypeError, "indices"),
            (dict(top=(v.half(), i, r)), TypeError, "values"),
            (dict(top=(v, i, torch.zeros(4, 1))), ValueError, "rest"),
            (dict(top=(v, i, r.double())), TypeError, "rest"),
            (dict(weight=torch.ones(3)), ValueError, "weight"),
            (dict(weight=w.bfloat16()), TypeError, "weight"),
            (dict(weight=w.clone().requires_grad_(True)), ValueError, "detach"),
            (dict(top=(v.clone().requires_grad_(True), i, r)), ValueError, "detach"),
            (dict(temperature=0.0), ValueError, "temperature"),
            (dict(reduction="batchmean"), ValueError, "reduction"),
            (dict(scale=float("nan")), ValueError, "scale"),
            (dict(logits=torch.zeros(1, 1025, 2), top=(torch.zeros(1, 3, 2), torch.zeros(1, 3, 2, dtype=torch.int64)),
                  weight=None), ValueError, "at most 1024"),
            (dict(), RuntimeError, "no CPU fallback")]:
        with pytest.raises(err, match=msg):
            ugpg.distillation_loss(**{**good, **kw})
    with pytest.raises(ValueError, match="k must"):
        ugpg.DistillationLoss(0)
    with pytest.raises(ValueError, match="temperature"):
        ugpg.DistillationLoss(3, temperature=-2.0)


def test_c_entries_refuse_before_any_launch():
    from ugpg import _C
    lib, p = _C.lib, 0x1000  # never dereferenced on the host

    def top(x=p, dt=0, N=4, V=9, inner=1, stride=9, k=3, T=1.0, v=p, i=p, r=p):
        return lib.ugpg_top_logits(x, dt, N, V, inner, stride, k, T, v, i, r, None)
    for kw in (dict(x=None), dict(x=p + 2), dict(dt=2), dict(N=0), dict(V=0), dict(inner=0), dict(stride=8),
               dict(k=0), dict(k=10), dict(V=999, stride=999, k=257), dict(T=0.0), dict(T=float("nan")),
               dict(v=None), dict(i=None), dict(r=None), dict(N=1 << 23), dict(inner=4, stride=9),
               dict(inner=1 << 31, stride=9 << 31), dict(V=(1 << 30) + 1, stride=1 << 31)):
        assert top(**kw) == -1, kw
        assert b"top_logits" in lib.ugpg_last_error()

    def desc(**kw):
        f = dict(logits=p, dtype=0, N=4, V=9, inner=1, stride=9, values=p, values_dtype=0, indices=p,
                 index_bits=64, k=3, rest=None, weight=None, temperature=1.0, scale=1.0)
        f.update(kw)
        return _C.DistillDesc(*f.values())
    for kw in (dict(logits=None), dict(dtype=3), dict(values=None), dict(indices=None), dict(values_dtype=2),
               dict(index_bits=16), dict(k=0), dict(temperature=-1.0),
               dict(temperature=1e-31), dict(temperature=2e30), dict(scale=float("nan")), dict(stride=3),
               dict(inner=2, V=1025, stride=2050, k=3)):
        d = desc(**kw)
        assert lib.ugpg_distill_workspace(C.byref(d), 0) == 0
        assert lib.ugpg_distill_fwd(C.byref(d), p, None, None, p, 1 << 30, None) == -1, kw
        assert lib.ugpg_distill_bwd(C.byref(d), p, 0, 0, p, p, 1 << 30, None) == -1, kw
        assert b"distill_bwd" in lib.ugpg_last_error()
    for kw in (dict(), dict(N=3, V=100000, stride=100000), dict(inner=100, stride=900)):
        d = desc(**kw)
        need, nb = (lib.ugpg_distill_workspace(C.byref(d), b) for b in (0, 1))
        assert need > 0 and (nb > 0) == (d.V > 512)
        assert lib.ugpg_distill_fwd(C.byref(d), p, None, None, p, need - 1, None) == -3
        assert lib.ugpg_distill_fwd(C.byref(d), p, None, None, None, need, None) == -3
        if nb:
            assert lib.ugpg_distill_bwd(C.byref(d), p, 0, 0, p, p, nb - 1, None) == -3
            assert lib.ugpg_distill_bwd(C.byref(d), p, 0, 0, p, None, nb, None) == -3
    d = desc(N=1 << 22, V=1 << 30, stride=1 << 30)  # more blocks than a grid takes
    assert lib.ugpg_distill_workspace(C.byref(d), 0) == 0
    d = desc()
    assert lib.ugpg_distill_fwd(C.byref(d), p, None, p + 2, p, 1 << 20, None) == -1
    assert lib.ugpg_distill_bwd(C.byref(d), p, 0, 0, p + 2, p, 1 << 20, None) == -1
    assert lib.ugpg_distill_fwd(C.byref(d), None, None, None, p, 1 << 20, None) == -1
    assert lib.ugpg_distill_bwd(C.byref(d), None, 0, 0, p, p, 1 << 20, None) == -1
    assert lib.ugpg_distill_bwd(C.byref(d), p, 0, 0, None, p, 1 << 20, None) == -1
    assert lib.ugpg_distill_bwd(C.byref(d), p, 1, 1, p, p, 1 << 20, None) == -1
