"""A teacher's top logits and the distillation loss against their definitions in 64 bits: every
kernel form (a wave a row, a block a row, a row split over blocks, a thread a pixel), both
types, ties, masks that leave a row little or nothing, absent and repeated entries.

Tolerances.  A sum of exponentials over a row is at most 64 float32 additions deep, an
exponent (z - m)/T carries 3 roundings of at most 126 (beyond that the term is below the
smallest float32): both stay below 2^-16 relative, 2^-15 together.  That is the error of every
probability, relative to itself, and (through the logarithm of the sum) of a row's KL,
absolutely.  A stored value adds half a step: 2^-24 of itself in float32, 2^-8 in bfloat16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
REL = 2.0 ** -15
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


# ------------------------------------------------------------------ definitions
def ref_top(logits, k, T):
    z = logits.double().movedim(1, -1)
    v, i = torch.sort(z, dim=-1, descending=True, stable=True)
    others = v[..., k:]
    rest = T * torch.logsumexp(others / T, -1) if others.shape[-1] else torch.full_like(v[..., 0], -math.inf)
    return v[..., :k].movedim(-1, 1), i[..., :k].movedim(-1, 1), rest


def ref_loss(logits, values, indices, rest, weight, T, scale):
    """-> per-row loss (lead shape), dlogits of their sum, and the bound's p + q part."""
    z = logits.detach().double().movedim(1, -1)
    lead, V = z.shape[:-1], z.shape[-1]
    z = z.reshape(-1, V)
    R = len(z)
    idx = indices.movedim(1, -1).reshape(R, -1).clone()
    val = values.double().movedim(1, -1).reshape(R, -1)
    k = idx.shape[1]
    idx[(idx < 0) | (idx >= V)] = -1
    for j in range(1, k) if k <= 16 else ():  # a repeated index counts once
        idx[:, j][(idx[:, :j] == idx[:, j:j + 1]).any(1)] = -1
    there = idx >= 0
    t = val.masked_fill(~there, -math.inf)
    r = (rest.double().reshape(R, 1) if rest is not None
         else torch.full((R, 1), -math.inf, dtype=torch.float64, device=z.device))
    tq = torch.cat([t, r], 1) / T
    says = tq.amax(1) > -math.inf
    says |= tq.isnan().any(1)
    q = torch.softmax(tq, 1)
    rows = torch.arange(R, device=z.device)[:, None].expand_as(idx)
    kept = torch.zeros_like(z, dtype=torch.bool)
    kept[rows[there], idx[there]] = True
    logp = torch.log_softmax(z / T, 1)
    lp_top = logp.gather(1, idx.clamp_min(0)).masked_fill(~there, -math.inf)
    lp_rest = torch.logsumexp(logp.masked_fill(kept, -math.inf), 1, keepdim=True)
    both = torch.cat([lp_top, lp_rest], 1)
    logq = torch.log_softmax(tq, 1)
    kl = torch.where(q > 0, q * (logq - both), torch.zeros_like(q)).sum(1)
    w = torch.ones_like(kl) if weight is None else weight.double().reshape(R)
    use = says & (w != 0)
    loss = torch.where(use, scale * T * T * w * kl, torch.zeros_like(kl))
    back = torch.where(lp_rest > -math.inf, (logp - lp_rest).exp(), torch.zeros_like(z)) * q[:, k:]
    back = back.masked_fill(kept, 0.0)
    back[rows[there], idx[there]] = q[:, :k][there]
    p = logp.exp()
    coef = torch.where(use, scale * T * w, torch.zeros_like(w))[:, None]
    dz = torch.where(use[:, None], coef * (p - back), torch.zeros_like(p))
    size = torch.where(use[:, None], coef.abs() * (p + back), torch.zeros_like(p))
    shape = lambda a: a.reshape(*lead, V).movedim(-1, 1)
    return loss.reshape(lead), shape(dz), shape(size), (scale * T * T * w * use).abs().reshape(lead)


def check_loss(got, rows, unit, count=1.0):
    """got against the rows' sum; unit: a row's loss per unit of KL."""
    want = rows.sum().item()
    lim = REL * unit.sum().item() + 2.0 ** -23 * abs(want)
    assert abs(got.item() - want) <= lim, (got.item(), want, lim)


def check_grad(got, dz, size):
    lim = REL * size + HALF[got.dtype] * dz.abs() + 1e-37
    err = (got.double() - dz).abs()
    bad = ~(err <= lim)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} gradients off; worst "
                           f"{(err / lim)[bad].max().item():.2f} times the bound")


def record(shape, k, dev, dtype, T, seed=0):
    """A student, and a teacher's record of it plus noise."""
    g = torch.Generator(device=dev).manual_seed(seed)
    teacher = (torch.randn(shape, generator=g, device=dev) * 2).to(dtype)
    student = (teacher.float() + torch.randn(shape, generator=g, device=dev)).to(dtype)
    v, i, r = ref_top(teacher, k, T)
    lead = (shape[0], *shape[2:])
    w = 0.5 + torch.rand(lead, generator=g, device=dev)
    return student, v.to(dtype).contiguous(), i.contiguous(), r.float(), w


# ------------------------------------------------------------------ top logits
TOP_SHAPES = [((1, 1), 1), ((3, 7), 3), ((5, 64), 64), ((6, 65), 65), ((4, 100), 1), ((2, 512), 256),
              ((3, 513), 256), ((2, 1000), 20), ((2, 2048), 256), ((2, 2049), 200), ((3, 5000), 64),
              ((2, 16385), 128), ((2, 50003), 20), ((1, 131072), 256), ((1, 300001), 50),
              ((300, 130), 17), ((2, 1, 3, 5), 1), ((2, 8, 5, 7), 3), ((1, 16, 9, 31), 16),
              ((2, 30, 4, 4), 8), ((1, 33, 6, 7), 33), ((2, 200, 3, 3), 60), ((3, 12, 17), 5)]


def fill(kind, shape, dev, dtype, seed=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    z = torch.randn(shape, generator=g, device=dev) * 3
    V = shape[1]
    pos = torch.arange(V, device=dev).view(1, V, *[1] * (len(shape) - 2)).float()
    low = torch.finfo(dtype).min
    if kind == "equal":
        z = torch.full(shape, 1.5, device=dev)
    elif kind == "ascending":
        z = (pos / V).expand(shape).clone()
    elif kind == "ties":
        z = torch.randint(-2, 3, shape, generator=g, device=dev).float()
    elif kind == "zeros":
        z = torch.where(z > 0, 0.0, -0.0)
    elif kind == "masked":  # all but every 37th place
        z = torch.where(pos % 37 == 5, z, -math.inf)
    elif kind == "lowest":
        z = torch.where(pos % 37 == 5, z, low)
    elif kind == "huge":  # products with log2(e)/T leave float32
        z = torch.where(pos % 5 == 2, 3e38, torch.where(pos % 5 == 3, -3e38, z))
    elif kind == "nothing":
        z = torch.full(shape, -math.inf, device=dev)
    elif kind == "inf":
        z = torch.where(pos % 11 == 3, math.inf, z)
    elif kind == "nan":
        z = torch.where(pos % 13 == 4, math.nan, z)
    elif kind == "one_nan":
        z = torch.where(pos == V // 2, math.nan, z)
    elif kind == "one_thread":  # the large values where one thread of 512 reads
        z = torch.where((pos % 4096 < 4) | (pos % 2048 < 4), z + 50, z)
    elif kind == "confident":
        z = torch.where(pos == V // 3, 80.0, z)
    return z.to(dtype)


KINDS = ["random", "equal", "ascending", "ties", "zeros", "masked", "lowest", "huge", "nothing", "inf", "nan",
         "one_nan", "one_thread", "confident"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_logits(dev, dtype, kind):
    import ugpg
    for shape, k in TOP_SHAPES:
        for T in (0.5, 1.0, 2.0) if kind in ("random", "lowest", "huge") else (1.5,):
            z = fill(kind, shape, dev, dtype)
            top = ugpg.teacher_top_logits(z, k, T)
            v, i, r = ref_top(z, k, T)
            assert top.values.dtype == dtype and top.indices.dtype == torch.int64
            assert top.values.shape == v.shape and top.rest.shape == r.shape
            assert torch.equal(top.indices, i), (shape, k)
            assert torch.equal(top.values.double().nan_to_num(7e7), v.nan_to_num(7e7)), (shape, k)
            same = (top.rest.double() == r) | (top.rest.isnan() & r.isnan())
            # a rest near the type's lowest value leaves float32 only at the last step
            lim = T * REL + 2.0 ** -23 * r.abs()
            ok = same | ((top.rest.double() - r).abs() <= lim)
            assert ok.all(), (shape, k, top.rest[~ok][:3], r[~ok][:3])


@pytest.mark.parametrize("V", [66, 127, 255, 257, 511, 513, 769, 1000, 1023, 1025, 1100, 2000, 2047, 3001])
def test_top_logits_of_middling_rows(dev, V):
    """A wave a row up to 1024 classes, then a block whose vectors may be fewer than the entries;
    rows that begin and end anywhere."""
    import ugpg
    for kind in ("random", "ties", "equal", "masked", "nan", "one_nan", "nothing", "zeros"):
        for dtype in (F32, BF16):
            z = fill(kind, (9, V + 3), dev, dtype, seed=V)[:, 1:V + 1]
            for k in sorted({1, 2, 63, 64, 65, 250, 256} | {V if V <= 256 else 200}):
                if k > V:
                    continue
                top = ugpg.teacher_top_logits(z, k, 1.5)
                v, i, r = ref_top(z, k, 1.5)
                assert torch.equal(top.indices, i), (kind, k)
                assert torch.equal(top.values.double().nan_to_num(7e7), v.nan_to_num(7e7)), (kind, k)
                same = (top.rest.double() == r) | (top.rest.isnan() & r.isnan())
                assert (same | ((top.rest.double() - r).abs() <= 1.5 * REL + 2.0 ** -23 * r.abs())).all(), (kind, k)


@pytest.mark.parametrize("shape,k", [((2, 20, 300, 240), 6), ((2, 24, 270, 250), 20), ((1, 100, 37, 41), 2),
                                     ((3, 70, 8, 9), 4), ((1, 1000, 5, 13), 5), ((1, 5000, 3, 5), 9),
                                     ((1, 35, 1, 2), 35)])
def test_top_logits_of_maps(dev, shape, k):
    """One thread or four a pixel, one reading or several."""
    import ugpg
    for kind in ("random", "ties", "equal", "ascending", "masked", "nan", "inf"):
        z = fill(kind, shape, dev, F32 if kind != "ties" else BF16, seed=5)
        top = ugpg.teacher_top_logits(z, k, 1.5)
        v, i, r = ref_top(z, k, 1.5)
        assert torch.equal(top.indices, i), kind
        assert torch.equal(top.values.double().nan_to_num(7e7), v.nan_to_num(7e7)), kind
        same = (top.rest.double() == r) | (top.rest.isnan() & r.isnan())
        assert (same | ((top.rest.double() - r).abs() <= 1.5 * REL + 2.0 ** -23 * r.abs())).all(), kind


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,k", [((2, 16, 19, 21), 12), ((1, 40, 65, 3), 5), ((3, 257, 7, 11), 100),
                                     ((1, 1024, 3, 23), 256), ((2, 64, 128, 128), 8)])
def test_loss_of_maps_in_parts(dev, shape, k, dtype):
    """Four threads a pixel; entries absent, repeated, and rows without weight among them."""
    import ugpg
    z, v, i, r, w = record(shape, k, dev, dtype, 2.0, seed=k)
    i = i.clone()
    i[:, 1, ::2] = -1
    if k <= 16:
        i[:, 3, :, ::3] = i[:, 0, :, ::3]
    w = w.clone()
    w[..., ::5] = 0.0
    rows, dz, size, unit = ref_loss(z, v, i, r, w, 2.0, 1.0)
    zr = z.clone().requires_grad_(True)
    loss = ugpg.distillation_loss(zr, (v, i, r), 2.0, weight=w, reduction="sum")
    check_loss(loss, rows, unit)
    loss.backward()
    check_grad(zr.grad, dz, size)
    out = ugpg.distillation_loss(z, (v, i, r), 2.0, weight=w, reduction="none")
    assert ((out.double() - rows).abs() <= REL * unit + 2.0 ** -23 * rows.abs()).all()


def test_top_logits_strides_and_alignment(dev):
    import ugpg
    for dtype in (F32, BF16):
        wide = fill("random", (5, 3001), dev, dtype)
        for z in (wide[:, :2500], wide[:, 1:2600], wide[1:, 3:], wide[::2, :2999], wide.t()[:700].t(),
                  wide[:1].expand(3, -1)):
            top = ugpg.teacher_top_logits(z, 37)
            v, i, r = ref_top(z, 37, 1.0)
            assert torch.equal(top.indices, i) and torch.equal(top.values.double(), v)
            assert ((top.rest.double() - r).abs() <= REL + 2.0 ** -23 * r.abs()).all()


def test_top_logits_same_bits_every_time(dev):
    import ugpg
    for kind in ("random", "ties", "masked"):
        z = fill(kind, (7, 40001), dev, BF16)
        first = ugpg.teacher_top_logits(z, 100)
        for _ in range(4):
            again = ugpg.teacher_top_logits(z, 100)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


# ------------------------------------------------------------------ the loss
LOSS_SHAPES = [((1, 2), 1), ((16, 7), 3), ((64, 64), 64), ((65, 65), 20), ((3, 512), 256), ((130, 500), 33),
               ((2, 513), 10), ((300, 513), 256), ((257, 1000), 7), ((2, 5000), 64), ((300, 4099), 50),
               ((256, 9001), 100), ((3, 50003), 20), ((1, 131072), 256), ((1, 270001), 30),
               ((2, 2, 3, 5), 1), ((2, 8, 15, 17), 3), ((1, 33, 9, 31), 8), ((1, 1024, 2, 3), 40), ((3, 12, 17), 5)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,k", LOSS_SHAPES)
def test_loss_and_gradient(dev, shape, k, dtype):
    import ugpg
    for T, with_rest, with_w in ((2.0, True, True), (1.0, False, False), (0.5, True, False)):
        z, v, i, r, w = record(shape, k, dev, dtype, T, seed=k)
        r, w = (r if with_rest else None), (w if with_w else None)
        n = z.numel() // shape[1]
        rows, dz, size, unit = ref_loss(z, v, i, r, w, T, 1.0 / n)
        zr = z.clone().requires_grad_(True)
        loss = ugpg.distillation_loss(zr, ugpg.TopLogits(v, i, r), T, weight=w)
        assert loss.dtype == F32 and loss.dim() == 0
        check_loss(loss, rows, unit)
        (g,) = torch.autograd.grad(loss, (zr,))
        assert g.dtype == dtype and g.shape == z.shape
        check_grad(g, dz, size)
        with torch.no_grad():  # the same loss without a gradient
            quiet = ugpg.distillation_loss(z, (v, i, r), T, weight=w)
        assert torch.equal(quiet, loss.detach())


@pytest.mark.parametrize("shape,k", [((16, 7), 3), ((130, 100), 9), ((3, 9001), 20), ((260, 3000), 20),
                                     ((2, 8, 6, 7), 3)])
def test_reductions_scales_and_upstream_gradients(dev, shape, k):
    import ugpg
    z, v, i, r, w = record(shape, k, dev, F32, 1.5, seed=3)
    n = z.numel() // shape[1]
    top = ugpg.TopLogits(v, i.int(), r)
    lead = (shape[0], *shape[2:])
    g = torch.Generator(device=dev).manual_seed(1)
    up = torch.randn(lead, generator=g, device=dev)
    rows, dz, size, unit = ref_loss(z, v, i, r, w, 1.5, 1.0)
    for red, scale, s in (("sum", 1.0, 1.0), ("mean", 1.0, 1.0 / n), ("mean", 0.25, 0.25 / n), ("sum", -2.0, -2.0)):
        for factor in (1.0, 3.0, 0.0):
            zr = z.clone().requires_grad_(True)
            loss = ugpg.distillation_loss(zr, top, 1.5, weight=w, reduction=red, scale=scale)
            check_loss(loss, rows * s, unit * abs(s))
            (factor * loss).backward()
            check_grad(zr.grad, dz * (s * factor), size * abs(s * factor))
    zr = z.clone().requires_grad_(True)
    out = ugpg.distillation_loss(zr, top, 1.5, weight=w, reduction="none")
    assert out.shape == lead
    assert ((out.double() - rows).abs() <= REL * unit + 2.0 ** -23 * rows.abs()).all()
    (out * up).sum().backward()
    u = up.double().unsqueeze(1)
    check_grad(zr.grad, dz * u, size * u.abs())


def test_second_backward_and_shared_logits(dev):
    """retain_graph: the gradient handed out first is not touched by the second pass; the
    logits feed another loss as well."""
    import ugpg
    z, v, i, r, w = record((40, 3000), 16, dev, F32, 2.0)
    zr = z.clone().requires_grad_(True)
    loss = ugpg.distillation_loss(zr, (v, i, r), 2.0)
    (a,) = torch.autograd.grad(loss, (zr,), retain_graph=True)
    keep = a.clone()
    (b,) = torch.autograd.grad(2.0 * loss, (zr,), retain_graph=True)
    (c,) = torch.autograd.grad(loss, (zr,))
    assert torch.equal(a, keep) and torch.equal(c, keep)
    _, dz, size, _ = ref_loss(z, v, i, r, None, 2.0, 1.0 / 40)
    check_grad(b, 2 * dz, 2 * size)
    other = (zr * 0.5).sum() + ugpg.distillation_loss(zr, (v, i, r), 2.0)
    (d,) = torch.autograd.grad(other, (zr,))
    assert torch.equal(d, keep + 0.5)


@pytest.mark.parametrize("shape,k", [((20, 9), 4), ((70, 300), 6), ((3, 9001), 12), ((260, 1500), 6),
                                     ((2, 12, 5, 6), 4)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_absent_repeated_and_empty(dev, shape, k, dtype):
    """Entries of index -1, far outside, and repeated; rows without any entry, with and without
    a rest; rows of weight 0 that hold NaN; a teacher's row of -inf."""
    import ugpg
    z, v, i, r, w = record(shape, k, dev, dtype, 1.0, seed=11)
    V = shape[1]
    i[0, 1] = -1
    v[0, 1] = math.nan
    i[0, 2] = V
    v[0, 2] = math.inf
    i[1, k - 1] = i[1, 0]
    if len(shape) == 2:
        v[2], i[2] = math.nan, -1          # nothing but the rest
        z2 = z.clone()
        if shape[0] > 3:
            w[3] = 0.0
            z2[3] = math.nan
            v[4], r[4] = -math.inf, -math.inf
            i[5] = 2 ** 40
    else:
        v[1, :, 2, 3], i[1, :, 2, 3] = math.nan, -1
        w[0, 1, 1] = 0.0
        z2 = z.clone()
        z2[0, :, 1, 1] = math.nan
    for rest in (r, None):
        rows, dz, size, unit = ref_loss(z, v, i, rest, w, 1.0, 1.0)
        zr = z2.clone().requires_grad_(True)
        loss = ugpg.distillation_loss(zr, (v, i, rest), 1.0, weight=w, reduction="sum")
        check_loss(loss, rows, unit)
        loss.backward()
        check_grad(zr.grad, dz, size)
    nothing = torch.full_like(i, -1)
    zr = z.clone().requires_grad_(True)
    loss = ugpg.distillation_loss(zr, (v, nothing, None))
    loss.backward()
    assert loss.item() == 0.0 and not zr.grad.any()


@pytest.mark.parametrize("shape,k", [((9, 40), 5), ((66, 40), 5), ((4, 9001), 20), ((258, 700), 5), ((1, 10, 4, 5), 3)])
def test_masked_students(dev, shape, k):
    """Student logits of -inf, of the type's lowest value, and far apart, outside and inside the
    record; k = V (an empty rest); what cannot be learned is an infinite loss, never NaN."""
    import ugpg
    z, v, i, r, w = record(shape, k, dev, F32, 0.5, seed=13)
    out = torch.ones_like(z, dtype=torch.bool).scatter_(1, i, False)
    g = torch.Generator(device=dev).manual_seed(2)
    some = out & (torch.rand(z.shape, generator=g, device=dev) < 0.5)
    for bad in (-math.inf, torch.finfo(F32).min, -1000.0):
        zb = torch.where(some, bad, z)
        rows, dz, size, unit = ref_loss(zb, v, i, r, None, 0.5, 1.0)
        zr = zb.clone().requires_grad_(True)
        loss = ugpg.distillation_loss(zr, (v, i, r), 0.5, reduction="sum")
        check_loss(loss, rows, unit)
        loss.backward()
        check_grad(zr.grad, dz, size)
    # everything outside the record at the type's lowest value, or beyond what T divides
    for bad in (torch.finfo(F32).min, 3e38):
        zb = torch.where(out, bad, z)
        rows, dz, size, unit = ref_loss(zb, v, i, None, None, 0.5, 1.0)
        zr = zb.clone().requires_grad_(True)
        loss = ugpg.distillation_loss(zr, (v, i, None), 0.5, reduction="sum")
        loss.backward()
        if bad < 0:
            check_loss(loss, rows, unit)
        check_grad(zr.grad, dz, size)
    # all others masked: with no rest in the record that is fine, with one it is infinite
    zb = torch.where(out, -math.inf, z)
    rows, dz, size, unit = ref_loss(zb, v, i, None, None, 0.5, 1.0)
    zr = zb.clone().requires_grad_(True)
    loss = ugpg.distillation_loss(zr, (v, i, None), 0.5, reduction="sum")
    check_loss(loss, rows, unit)
    loss.backward()
    check_grad(zr.grad, dz, size)
    zr = zb.clone().requires_grad_(True)
    loss = ugpg.distillation_loss(zr, (v, i, r), 0.5, reduction="sum")
    assert loss.item() == math.inf
    loss.backward()
    assert zr.grad.isfinite().all() and not zr.grad[out].any()
    # a kept class masked in the student
    zb = z.clone()
    zb.scatter_(1, i[:, :1], -math.inf)
    zr = zb.clone().requires_grad_(True)
    loss = ugpg.distillation_loss(zr, (v, i, r), 0.5, reduction="sum")
    loss.backward()
    _, dz, size, _ = ref_loss(zb, v, i, r, None, 0.5, 1.0)
    assert loss.item() == math.inf
    check_grad(zr.grad, dz, size)


def test_confident_rows_keep_their_rest(dev):
    """Nearly all mass in the record on both sides: the rest's share (e^-30) survives, where a
    total minus the kept classes would leave nothing of it."""
    import ugpg
    for shape in ((4, 50), (4, 9000), (300, 800)):
        g = torch.Generator(device=dev).manual_seed(4)
        z = torch.randn(shape, generator=g, device=dev)
        t = torch.randn(shape, generator=g, device=dev)
        z[:, 7] = 40.0
        t[:, 7] = 38.0
        top = ugpg.teacher_top_logits(t, 1, 1.0)
        assert (top.rest < 12).all()
        zr = z.clone().requires_grad_(True)
        loss = ugpg.distillation_loss(zr, top, 1.0, reduction="sum")
        loss.backward()
        rows, dz, size, unit = ref_loss(z, top.values, top.indices, top.rest, None, 1.0, 1.0)
        check_loss(loss, rows, unit)
        rest = torch.ones(shape[1], dtype=torch.bool, device=dev)
        rest[7] = False
        # relative to each probability: this is the point
        check_grad(zr.grad[:, rest], dz[:, rest], size[:, rest])
        assert (dz[:, rest] != 0).all() and (zr.grad[:, rest] != 0).all()


def test_many_short_rows(dev):
    """More rows than the waves in flight: every block steps over several."""
    import ugpg
    for shape, k in (((200003, 7), 3), ((140001, 33), 5)):
        z, v, i, r, w = record(shape, k, dev, F32, 2.0, seed=19)
        rows, dz, size, unit = ref_loss(z, v, i, r, w, 2.0, 1.0 / shape[0])
        zr = z.clone().requires_grad_(True)
        loss = ugpg.distillation_loss(zr, (v, i, r), 2.0, weight=w)
        check_loss(loss, rows, unit)
        loss.backward()
        check_grad(zr.grad, dz, size)
        out = ugpg.distillation_loss(z, (v, i, r), 2.0, weight=w, reduction="none")
        assert ((out.double() - rows * shape[0]).abs() <= REL * unit * shape[0] + 2.0 ** -23 * out.double().abs()).all()


def test_strides_alignment_and_mixed_types(dev):
    import ugpg
    for dtype in (F32, BF16):
        wide = fill("random", (300, 1203), dev, dtype, seed=5)
        for z in (wide[:, :1000], wide[:, 1:1100], wide[:5, 3:], wide.t()[:700].t(), wide[::3, 2:900]):
            V = z.shape[1]
            v, i, r = ref_top(z.float() + 0.5 * fill("random", z.shape, dev, F32, 6), 12, 1.0)
            for vals in (v.float(), v.to(BF16)):
                zr = z.detach().requires_grad_(True)
                loss = ugpg.distillation_loss(zr, (vals, i.int(), r.float()), 1.0)
                (g,) = torch.autograd.grad(loss, (zr,))
                rows, dz, size, unit = ref_loss(z, vals, i, r.float(), None, 1.0, 1.0 / z.shape[0])
                check_loss(loss, rows, unit)
                check_grad(g, dz, size)


@pytest.mark.parametrize("shape,k", [((20, 9), 4), ((70, 300), 6), ((3, 9001), 12), ((260, 1501), 6),
                                     ((2, 12, 5, 6), 4)])
def test_writes_stay_inside(dev, shape, k):
    import ctypes as C
    import ugpg
    from tests._guard import guarded
    from ugpg import _C, ops
    for dtype in (F32, BF16):
        z, v, i, r, w = record(shape, k, dev, dtype, 2.0)
        N, V = shape[:2]
        inner = z.numel() // (N * V)
        stride, code = V * inner, ops._dtype_code(z)
        d = _C.DistillDesc(z.data_ptr(), code, N, V, inner, stride, v.data_ptr(), code, i.data_ptr(), 64, k,
                           r.data_ptr(), w.data_ptr(), 2.0, 1.0)
        need = _C.lib.ugpg_distill_workspace(C.byref(d), 0)
        work = guarded((need,), dev, torch.uint8)
        loss, rows = guarded((1,), dev), guarded((z.numel() // shape[1],), dev)
        dz = guarded(shape, dev, dtype)
        _C.check(_C.lib.ugpg_distill_fwd(C.byref(d), loss.t.data_ptr(), rows.t.data_ptr(), dz.t.data_ptr(),
                                         work.t.data_ptr(), need, ops.stream()), "distill_fwd")
        for n, t in (("ws", work), ("loss", loss), ("rows", rows), ("dlogits", dz)):
            t.check(n)
        zr = z.clone().requires_grad_(True)
        want = ugpg.distillation_loss(zr, (v, i, r), 2.0, weight=w, reduction="sum")
        (grad,) = torch.autograd.grad(want, (zr,))
        assert torch.equal(want.detach().view(1), loss.t) and torch.equal(grad, dz.t)
        # a partial record's buffers too
        vals, idx, rest = guarded(v.shape, dev, dtype), guarded((2 * i.numel(),), dev, torch.int32), guarded(r.shape, dev)
        _C.check(_C.lib.ugpg_top_logits(z.data_ptr(), code, N, V, inner, stride, k, 2.0,
                                        vals.t.data_ptr(), idx.t.data_ptr(), rest.t.data_ptr(), ops.stream()), "top")
        for n, t in (("values", vals), ("indices", idx), ("rest", rest)):
            t.check(n)


@pytest.mark.parametrize("shape,k", [((20, 9), 4), ((3, 9001), 12), ((260, 1501), 6), ((2, 12, 5, 6), 4)])
def test_gradient_against_differences(dev, shape, k):
    """Along the gradient's own direction u, step h = 1/4 / max|u|: the loss's third derivative is
    below its gradient's size, so h^2/6 of it bounds the difference quotient's error, and 2^-15
    of the loss over the step bounds rounding's: 2 % covers both."""
    import ugpg
    z, v, i, r, w = record(shape, k, dev, F32, 2.0, seed=17)
    f = lambda t: ugpg.distillation_loss(t, (v, i, r), 2.0, weight=w, reduction="none").double().sum()
    zr = z.clone().requires_grad_(True)
    ugpg.distillation_loss(zr, (v, i, r), 2.0, weight=w, reduction="sum").backward()
    u = zr.grad
    h = 0.25 / u.abs().max().item()
    num = (f(z + h * u) - f(z - h * u)).item() / (2 * h)
    want = (u.double() ** 2).sum().item()
    assert abs(num - want) <= 0.02 * want


def test_other_stream_and_captured_graph(dev):
    import ugpg
    for shape, k in (((16, 7), 3), ((300, 1100), 8), ((2, 20000), 8), ((2, 8, 9, 9), 3)):
        z, v, i, r, w = record(shape, k, dev, F32, 2.0)
        teacher = fill("random", shape, dev, F32, 9)

        def step(x, t):
            top = ugpg.teacher_top_logits(t, k, 2.0)
            loss = ugpg.distillation_loss(x, top, 2.0, weight=w)
            return (*top, loss.detach(), *torch.autograd.grad(3.0 * loss, (x,)))
        leaf = lambda: z.clone().requires_grad_(True)
        want = [t.clone() for t in step(leaf(), teacher)]
        side = torch.cuda.Stream()
        x = leaf()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(x, teacher)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        x, t = leaf(), teacher.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(x, t)
        for n in range(3):
            with torch.no_grad():
                x.copy_(z * (1.0 + 0.5 * n))
                t.copy_(teacher * (1.0 - 0.25 * n))
            graph.replay()
            torch.cuda.synchronize()
            ex = step(x.detach().clone().requires_grad_(True), t.clone())
            assert all(torch.equal(a, b) for a, b in zip(outs, ex)), n


def test_capture_beside_a_living_eager_graph_is_refused(dev):
    import ugpg
    z, v, i, r, w = record((70, 33), 5, dev, F32, 2.0, seed=23)
    leaf = z.clone().requires_grad_(True)
    want = torch.autograd.grad(ugpg.distillation_loss(leaf, (v, i, r), 2.0), leaf)[0]
    alive = leaf * 1.0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="default stream"):
            ugpg.distillation_loss(leaf, (v, i, r), 2.0)
        still = ugpg.distillation_loss(leaf.detach(), (v, i, r), 2.0)
    del alive
    graph.replay()
    assert torch.isfinite(still)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ugpg.distillation_loss(leaf, (v, i, r), 2.0), leaf)[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_offsets_past_32_bits(dev):
    """Rows beyond 2^31 elements into the logits."""
    import ugpg
    N, V = 2100, 1 << 20
    z = torch.empty((N, V), dtype=BF16, device=dev).normal_()
    top = ugpg.teacher_top_logits(z[N - 2:], 20)
    full = ugpg.teacher_top_logits(z, 20)
    assert torch.equal(full.indices[N - 2:], top.indices) and torch.equal(full.values[N - 2:], top.values)
    zr = z.requires_grad_(True)
    loss = ugpg.distillation_loss(zr, full, 2.0, reduction="none")
    (g,) = torch.autograd.grad(loss.sum(), (zr,))
    rows, dz, size, unit = ref_loss(z[N - 2:].detach(), top.values, top.indices, full.rest[N - 2:], None, 2.0, 1.0)
    assert ((loss[N - 2:].double() - rows).abs() <= REL * unit + 2.0 ** -23 * rows.abs()).all()
    check_grad(g[N - 2:], dz, size)


def test_differentiable_once(dev):
    """Second derivatives are refused, not silently zero; create_graph alone is fine."""
    import ugpg
    z, v, i, r, w = record((30, 7), 3, dev, F32, 2.0)
    zr = z.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ugpg.distillation_loss(zr, (v, i, r), 2.0), (zr,), create_graph=True)
    (h,) = torch.autograd.grad(ugpg.distillation_loss(zr, (v, i, r), 2.0), (zr,))
    assert torch.equal(g.detach(), h)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


def test_record_written_after_the_forward_is_noticed(dev):
    import ugpg
    z, v, i, r, w = record((30, 7), 3, dev, F32, 2.0)
    zr = z.clone().requires_grad_(True)
    loss = ugpg.distillation_loss(zr, (v, i, r), 2.0, weight=w)
    v.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        (2 * loss).backward()


def test_loss_object(dev):
    import ugpg
    z, v, i, r, w = record((30, 7), 3, dev, F32, 2.0)
    teacher = fill("random", (30, 7), dev, F32, 3)
    crit = ugpg.DistillationLoss(3, temperature=2.0, scale=0.5)
    top = ugpg.teacher_top_logits(teacher, 3, 2.0)
    want = ugpg.distillation_loss(z, top, 2.0, weight=w, scale=0.5)
    assert torch.equal(crit(z, teacher, weight=w), want) and torch.equal(crit(z, top, weight=w), want)
    assert torch.equal(ugpg.DistillationLoss(20)(z, teacher), ugpg.DistillationLoss(7)(z, teacher))
