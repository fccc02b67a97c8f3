"""The distillation loss where the student has nearly learned its teacher, and the rest's logit of
very long rows, within bounds derived from the kernels' sums (tests/_distill_bounds.py)."""
import pytest
import torch

from tests import _distill_bounds as db

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def near(shape, k, dev, dtype, T, noise, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    t = (2.0 * torch.randn(shape, generator=g, device=dev)).to(dtype)
    z = (t.float() + noise * torch.randn(shape, generator=g, device=dev)).to(dtype)
    return z, db.record(t.movedim(1, -1), k, T)


# a wave a row (in one block, in many), a block a row, a row over several blocks
@pytest.mark.parametrize("shape,k", [((16, 7), 3), ((64, 300), 20), ((20000, 40), 5), ((300, 500), 64),
                                     ((300, 4097), 64), ((700, 20000), 16), ((3, 9001), 20), ((2, 131071), 256)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("noise", [0.0, 2e-3, 0.1])
def test_rows_near_their_teacher(dev, shape, k, dtype, noise):
    import ugpg
    for T in (1.0, 2.0):
        z, (v, i, r) = near(shape, k, dev, dtype, T, noise, seed=k)
        kl, klim, dz, dlim = db.oracle(z, v, i, r, T)
        want, lim = T * T * kl, T * T * klim + 2.0 ** -24 * (T * T * kl)
        rows = ugpg.distillation_loss(z, (v, i, r), T, reduction="none")
        assert ((rows.double() - want).abs() <= lim).all(), ((rows.double() - want).abs() / lim).max().item()
        zr = z.clone().requires_grad_(True)
        loss = ugpg.distillation_loss(zr, (v, i, r), T)
        assert abs(loss.item() - want.mean().item()) <= lim.mean().item() + 2.0 ** -24 * want.mean().item()
        (g,) = torch.autograd.grad(loss * shape[0], (zr,))
        # (the upstream factor shape[0] / shape[0] rounds once on each side)
        bound = dlim + (db.HALF[dtype] + 2.0 ** -23) * dz.abs()
        assert ((g.double() - dz).abs() <= bound).all(), ((g.double() - dz).abs() / bound).max().item()


# logits and record in registers, marks in LDS, four threads a pixel
@pytest.mark.parametrize("shape,k", [((2, 8, 64, 64), 3), ((2, 16, 31, 33), 8), ((1, 30, 40, 40), 8),
                                     ((2, 24, 40, 41), 12), ((2, 64, 32, 32), 8), ((1, 60, 31, 17), 16)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("noise", [0.0, 2e-3, 0.1])
def test_maps_near_their_teacher(dev, shape, k, dtype, noise):
    import ugpg
    T = 2.0
    z, (v, i, r) = near(shape, k, dev, dtype, T, noise, seed=k)
    flat = lambda t: t.reshape(-1, t.shape[-1])
    kl, _, _, _ = db.oracle(flat(z.movedim(1, -1)), flat(v), flat(i), r.reshape(-1), T)
    want = T * T * kl
    lim = T * T * (db.MAP + db.KLREL * kl) + 2.0 ** -24 * want
    top = (v.movedim(-1, 1), i.movedim(-1, 1), r)
    out = ugpg.distillation_loss(z, top, T, reduction="none").double().reshape(-1)
    assert ((out - want).abs() <= lim).all(), ((out - want).abs() / lim).max().item()
    loss = ugpg.distillation_loss(z, top, T)
    assert abs(loss.item() - want.mean().item()) <= lim.mean().item() + 2.0 ** -24 * want.mean().item()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,k", [(50003, 64), (300001, 50), ((1 << 21) + 7, 100)])
def test_rest_of_long_rows(dev, V, k, dtype):
    """A thread adds its share of a row one after the other, a vector at a time or, in the exact
    selection that ties and NaN lead to, a value at a time: V / 512 additions at most, then a tree
    and the exponents' roundings: S is off by (V / 512 + 64) 2^-24 of itself, the logit T log S by
    T times as much."""
    import ugpg
    g = torch.Generator(device=dev).manual_seed(V)
    for kind in ("random", "equal", "few values"):
        z = torch.randn(2, V, generator=g, device=dev) * 2.0
        if kind == "equal":
            z = torch.full_like(z, 0.75)
        elif kind == "few values":
            z = z.round().clamp(-2, 2)
        z = z.to(dtype)
        for T in (0.5, 2.0):
            top = ugpg.teacher_top_logits(z, k, T)
            v, i, _ = db.record(z, k, T)
            others = z.double().scatter(1, i, -torch.inf)
            rest = T * torch.logsumexp(others / T, 1)
            assert torch.equal(top.indices, i) and torch.equal(top.values, v)
            lim = T * (V / 512 + 64) * 2.0 ** -24 + 2.0 ** -23 * rest.abs()
            assert ((top.rest.double() - rest).abs() <= lim).all(), (kind, T)
