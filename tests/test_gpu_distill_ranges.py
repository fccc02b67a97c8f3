"""Logits and temperatures of every size: masks of -1e9 to the type's lowest value, large positive
logits, temperatures over the whole documented range, and values on both sides of every
magnitude at which the kernels change how they take an exponent.

The rest's logit is T log S + m with S off by REL = 2^-15 of itself (128 additions at most in these
rows, exponents of at most 126); a loss by REL of a unit of KL, a gradient by REL (p + q), as in
tests/test_gpu_distill.py; and half a step of what is stored."""
import math

import pytest
import torch

from tests.test_gpu_distill import check_grad, check_loss, ref_loss, ref_top

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
REL = 2.0 ** -15
# a wave a row (64, 512, 1024 classes), a block a row, class maps of one and four threads a pixel
FORMS = [((70, 50), 5), ((9, 300), 20), ((9, 900), 20), ((3, 5000), 64), ((2, 40001), 100),
         ((2, 12, 5, 7), 3), ((1, 80, 6, 5), 4)]
# the loss: a wave a row, a block a row, a row over several blocks, maps
LOSSES = [((16, 50), 5), ((70, 500), 20), ((300, 1500), 20), ((3, 9001), 20), ((2, 8, 5, 7), 3), ((1, 24, 5, 7), 12),
          ((1, 80, 6, 5), 4)]


def check_rest(top, z, k, T, what):
    v, i, r = ref_top(z, k, T)
    assert torch.equal(top.indices, i) and torch.equal(top.values.double(), v), what
    lim = T * REL + 2.0 ** -23 * r.abs()
    bad = ~((top.rest.double() == r) | ((top.rest.double() - r).abs() <= lim))
    assert not bad.any(), (what, top.rest[bad][:3].tolist(), r[bad][:3].tolist())


def masked(shape, k, dev, dtype, level, seed=1):
    """k confident classes a row, all others within a few units of `level`."""
    g = torch.Generator(device=dev).manual_seed(seed)
    z = level + torch.randn(shape, generator=g, device=dev)
    pos = torch.arange(shape[1], device=dev).view(1, -1, *[1] * (len(shape) - 2))
    z = torch.where(pos % (shape[1] // k) == 0, level + abs(level) + 5.0 + pos / shape[1], z)
    return z.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)


LEVELS = [-1e6, -1e9, -1e10, -1e12, -1e20, -1e30, -3.3e38, 1e6, 1e10, 1e15, 1e30]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("level", LEVELS)
def test_rest_of_masked_rows(dev, dtype, level):
    import ugpg
    for shape, k in FORMS:
        z = masked(shape, k, dev, dtype, level)
        for T in (0.25, 1.0, 8.0, 100.0):
            check_rest(ugpg.teacher_top_logits(z, k, T), z, k, T, (shape, T))


@pytest.mark.parametrize("T", [1e-30, 1e-20, 1e-12, 1e-9, 1e-6, 1e-3, 1e3, 1e6, 1e12, 1e30])
def test_rest_at_every_temperature(dev, T):
    import ugpg
    for shape, k in FORMS:
        g = torch.Generator(device=dev).manual_seed(3)
        z = 5.0 * torch.randn(shape, generator=g, device=dev) - 3.0
        check_rest(ugpg.teacher_top_logits(z, k, T), z, k, T, shape)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("bits", [10, 16, 19, 20, 21, 24, 30])
def test_rows_across_a_magnitude(dev, bits, sign):
    """Values within a few units of sign * T 2^bits ln 2 (an exponent of 2^bits), rising and falling,
    so that a thread's maximum crosses it in either direction."""
    import ugpg
    for shape, k in FORMS:
        for T in (1.0, 3.0):
            mid = sign * T * 2.0 ** bits * math.log(2.0)
            ramp = torch.linspace(-6.0 * T, 6.0 * T, shape[1], device=dev).view(1, -1, *[1] * (len(shape) - 2))
            for way in (1.0, -1.0):
                z = (mid + way * ramp).expand(shape).contiguous()
                check_rest(ugpg.teacher_top_logits(z, k, T), z, k, T, (shape, T, way))


@pytest.mark.parametrize("level", LEVELS)
def test_loss_of_masked_students(dev, level):
    """All classes outside the record at one far level, in the student and in the teacher."""
    import ugpg
    for shape, k in LOSSES:
        for T in (1.0, 8.0):
            z = masked(shape, k, dev, F32, level, seed=2)
            v, i, r = ref_top(masked(shape, k, dev, F32, level, seed=4), k, T)
            v, i, r = v.float().contiguous(), i.contiguous(), r.float()
            rows, dz, size, unit = ref_loss(z, v, i, r, None, T, 1.0)
            zr = z.clone().requires_grad_(True)
            loss = ugpg.distillation_loss(zr, (v, i, r), T, reduction="sum")
            check_loss(loss, rows, unit)
            loss.backward()
            check_grad(zr.grad, dz, size)


@pytest.mark.parametrize("bits", [10, 16, 19, 20, 21, 24])
def test_loss_across_a_magnitude(dev, bits):
    import ugpg
    for shape, k in LOSSES:
        g = torch.Generator(device=dev).manual_seed(bits)
        for sign in (1.0, -1.0):
            T = 2.0
            mid = sign * T * 2.0 ** bits * math.log(2.0)
            ramp = torch.linspace(-4.0 * T, 4.0 * T, shape[1], device=dev).view(1, -1, *[1] * (len(shape) - 2))
            z = mid + ramp + torch.randn(shape, generator=g, device=dev)
            v, i, r = ref_top(z - sign + torch.randn(shape, generator=g, device=dev), k, T)
            v, i, r = v.float().contiguous(), i.contiguous(), r.float()
            rows, dz, size, unit = ref_loss(z, v, i, r, None, T, 1.0)
            zr = z.clone().requires_grad_(True)
            loss = ugpg.distillation_loss(zr, (v, i, r), T, reduction="sum")
            check_loss(loss, rows, unit)
            loss.backward()
            check_grad(zr.grad, dz, size)


@pytest.mark.parametrize("T", [1e-20, 1e-12, 1e-9, 1e-6, 1e-3])
def test_loss_at_small_temperatures(dev, T):
    """Here a row's KL is a difference of logits over T: the loss is T^2 of it, whose error beside
    REL of a unit is a rounding of itself."""
    import ugpg
    for shape, k in LOSSES:
        g = torch.Generator(device=dev).manual_seed(9)
        z = torch.randn(shape, generator=g, device=dev)
        v, i, r = ref_top(z + 0.5 * torch.randn(shape, generator=g, device=dev), k, T)
        v, i, r = v.float().contiguous(), i.contiguous(), r.float()
        rows, dz, size, unit = ref_loss(z, v, i, r, None, T, 1.0)
        zr = z.clone().requires_grad_(True)
        loss = ugpg.distillation_loss(zr, (v, i, r), T, reduction="sum")
        check_loss(loss, rows, unit)
        loss.backward()
        check_grad(zr.grad, dz, size)


@pytest.mark.parametrize("shape,k", [((2, 8, 5, 7), 3), ((1, 16, 5, 7), 8), ((1, 30, 4, 6), 8), ((1, 24, 5, 7), 12),
                                     ((1, 30, 3, 5), 24), ((1, 80, 6, 5), 4), ((1, 80, 4, 5), 40), ((70, 50), 5),
                                     ((3, 9001), 20)])
@pytest.mark.parametrize("bits", [90, 120, 128, 135, 145])
def test_lowest_logit_against_a_small_probability(dev, shape, k, bits):
    """A class the teacher keeps at 2^-bits, or its rest at 2^-bits, and the student at the type's lowest
    value: T^2 times 2^-bits times 3.4e38 / T is most of the loss or a visible part of it.  The exponent
    (t - M) c, of size `bits`, carries three roundings (the difference, c, the product), 2^-24 of it each,
    so its exponential is off by 3 bits ln 2 half steps of 2^-24, and 8 more for the exponential itself
    and the sums; the other terms by REL (rows) or 2^-19 (maps) of the unit."""
    import ugpg
    g = torch.Generator(device=dev).manual_seed(bits)
    low = torch.finfo(F32).min
    for T in (1.0, 3.0):
        t = 0.5 * torch.randn(shape, generator=g, device=dev)
        t[:, :k - 1] += 20.0 * T * math.log(2.0)
        t[:, k - 1] = t[:, 0] - bits * T * math.log(2.0)
        for far_rest in (False, True):
            z = t + 0.1 * torch.randn(shape, generator=g, device=dev)
            v, i = t[:, :k].clone(), torch.arange(k, device=dev).view(1, k, *[1] * (t.dim() - 2)).expand_as(t[:, :k])
            r = torch.full_like(t[:, 0], -math.inf)
            if far_rest:
                v[:, k - 1] = t[:, 0] - 1.0
                z[:, k:] = low
                r = t[:, 0] - bits * T * math.log(2.0)
            else:
                z[:, k - 1] = low
            i = i.contiguous()
            rows, _, _, unit = ref_loss(z, v, i, r, None, T, 1.0)
            out = ugpg.distillation_loss(z, (v, i, r), T, reduction="none")
            lim = (3 * bits * math.log(2.0) + 8) * 2.0 ** -24 * rows.abs() + (REL if z.dim() == 2 else 2.0 ** -19) * unit + 1e-30
            ok = ((out.double() - rows).abs() <= lim) | ((rows > 3.4e38) & (out == math.inf))
            assert ok.all(), (T, far_rest, out[~ok][:3].tolist(), rows[~ok][:3].tolist())
