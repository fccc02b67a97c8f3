"""Group normalisation with an activation against its definition in 64 bits: both forms of
the kernels (a slab resident in a block, two passes over chunks), every vector width, odd and
ragged sizes, both types, and the gradients against the formula's and against differences.

Tolerances: a value passes through a handful of float32 roundings (2^-24 each, relative to
the largest term), and its mean and rstd through sums whose error is at most 32 roundings
of the largest |x| (runs of 8, then trees): EPS32 = 48 * 2^-24 covers both against
scale = max|term| * (1 + max|x| * rstd).  A bfloat16 result adds half a step, 2^-8 of itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS32 = 48 * 2.0 ** -24
HALF16 = 2.0 ** -8


def ref(x, G, w, b, eps, act, dy=None):
    """64-bit definition; returns y, or (y, dx, dw, db, rstd)."""
    x = x.detach().double().requires_grad_(dy is not None)
    B, C = x.shape[0], x.shape[-1]
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    w.requires_grad_(True)
    b.requires_grad_(True)
    xg = x.reshape(B, -1, G, C // G)
    mean = xg.mean((1, 3), keepdim=True)
    rstd = ((xg - mean) ** 2).mean((1, 3), keepdim=True).add(eps).rsqrt()
    p = ((xg - mean) * rstd).reshape(x.shape) * w + b
    y = {"relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t), "none": lambda t: t}[act](p)
    if dy is None:
        return y.detach(), rstd.detach()
    gs = torch.autograd.grad(y, (x, w, b), dy.double())
    return (y.detach(), *gs, rstd.detach())


def off_corner(x, G, w, b, eps):
    """Move values whose pre-activation lies within 1e-3 of the ReLU's corner away from it:
    which side they fall on is a matter of rounding."""
    B, C = x.shape[0], x.shape[-1]
    xd = x.double().reshape(B, -1, G, C // G)
    mean = xd.mean((1, 3), keepdim=True)
    std = ((xd - mean) ** 2).mean((1, 3), keepdim=True).add(eps).sqrt()
    wv = w.double().view(1, 1, G, -1)
    p = (xd - mean) / std * wv + b.double().view(1, 1, G, -1)
    move = torch.where(p < 0, -1.0, 1.0) * 0.05 * std / wv
    return torch.where(p.abs() < 1e-3, xd + move, xd).reshape(x.shape).to(x.dtype)


def make(shape, G, dev, dtype, act, seed=0, offset=0.5, affine=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    C = shape[-1]
    x = torch.randn(shape, generator=g, device=dev) + offset * torch.randn(C, generator=g, device=dev)
    w = 0.5 + torch.rand(C, generator=g, device=dev)
    b = 0.3 * torch.randn(C, generator=g, device=dev)
    x = x.to(dtype)
    if act == "relu":
        x = off_corner(x, G, w, b, 1e-5)
    dy = torch.randn(shape, generator=g, device=dev).to(dtype)
    return x, (w if affine else None), (b if affine else None), dy


def near(got, want, scale, what, half=0.0):
    err = (got.double() - want).abs()
    lim = EPS32 * scale + half * want.abs()
    bad = (err > lim)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{(err - lim).max().item():.3e} over {EPS32 * scale:.3e}")


SHAPES = [
    # shape, groups: what it reaches
    ((1, 1, 1, 4), 2),            # one pixel, two channels a group
    ((3, 1, 1, 7), 7),            # one value a group: variance 0
    ((1, 16, 16, 512), 32),       # resident, 64-byte slabs
    ((16, 16, 16, 512), 32),      # resident, 128-byte slabs
    ((2, 64, 64, 256), 8),        # resident, 1024 threads (forward)
    ((2, 5, 3, 60), 12),          # resident, 5 channels a group: scalar accesses
    ((2, 9, 7, 36), 3),           # 12 channels a group, ragged rows
    ((1, 4, 4, 1024), 1),         # one group over everything
    ((1, 2, 2, 2048), 1),         # more channels than a resident block sums
    ((2, 40, 33, 64), 32),        # two channels a group
    ((2, 128, 96, 64), 32),       # two passes
    ((1, 200, 211, 7), 7),        # two passes, odd channels: scalar
    ((3, 75, 53, 60), 12),        # two passes, 4-wide
    ((1, 130, 128, 320), 4),      # two passes, 80 vector columns
    ((1, 70, 70, 1030), 5),       # two passes, several column blocks
    ((5, 33), 3),                 # no pixel axis at all
    ((2, 3, 4, 5, 24), 6),        # a three-dimensional image
]


@pytest.mark.parametrize("act", ["relu", "silu", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", SHAPES)
def test_forward_and_gradients(dev, shape, G, dtype, act):
    import ugpg
    x, w, b, dy = make(shape, G, dev, dtype, act)
    half = HALF16 if dtype == torch.bfloat16 else 0.0
    xr, wr, br = (t.clone().requires_grad_(True) for t in (x, w, b))
    y = ugpg.group_norm_act(xr, G, wr, br, 1e-5, act)
    dx, dw, db = torch.autograd.grad(y, (xr, wr, br), dy)
    ey, edx, edw, edb, rstd = ref(x, G, w, b, 1e-5, act, dy)
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == db.dtype == torch.float32
    r = rstd.max().item()
    cond = 1.0 + x.double().abs().max().item() * r
    near(y, ey, cond * ey.abs().max().clamp_min(1.0).item(), "y", half)
    n_g = x[0].numel() // G
    # dx: rstd times three terms of size |dy w|, |xh| of them; a group's constant part cancels
    sc = cond * r * 1.2 * (dy.double().abs().max() * w.double().max() * 4).item()
    near(dx, edx, sc * (1.0 + min(n_g, 64) ** 0.5), "dx", half)
    # sums over a batch's pixels: errors add like the terms' absolute values
    xh = 1.0 + x.double().abs().max().item() * r if n_g > 1 else 1.0
    terms = dy.double().abs().reshape(-1, shape[-1]).sum(0).max().item() * 1.2
    near(db, edb, cond * terms, "dbeta")
    near(dw, edw, cond * terms * xh, "dgamma")


@pytest.mark.parametrize("shape,G", [((2, 12, 10, 64), 8), ((2, 128, 96, 64), 32)])
def test_without_affine(dev, shape, G):
    import ugpg
    x, _, _, dy = make(shape, G, dev, torch.float32, "silu", affine=False)
    xr = x.clone().requires_grad_(True)
    y = ugpg.group_norm_act(xr, G, activation="silu")
    (dx,) = torch.autograd.grad(y, (xr,), dy)
    ey, edx, _, _, rstd = ref(x, G, None, None, 1e-5, "silu", dy)
    near(y, ey, 32.0, "y")
    near(dx, edx, 256.0 * rstd.max().item(), "dx")


@pytest.mark.parametrize("shape,G", [((2, 16, 16, 128), 8), ((1, 160, 128, 64), 32)])
def test_large_offset_keeps_the_variance(dev, shape, G):
    """mean/std = 1000: sum of squares minus the squared sum would lose the variance; the
    error allowed is that of x - mean in float32, 2^-24 * mean/std a rounding."""
    import ugpg
    g = torch.Generator(device=dev).manual_seed(3)
    x = 1000.0 + torch.randn(shape, generator=g, device=dev)
    y = ugpg.group_norm_act(x, G, activation="none")
    ey, _ = ref(x, G, None, None, 1e-5, "none")
    near(y, ey, 1000.0, "y")


@pytest.mark.parametrize("shape,G", [((2, 8, 6, 48), 4), ((2, 128, 96, 64), 8)])
@pytest.mark.parametrize("act", ["relu", "silu", "none"])
def test_gradient_against_differences(dev, shape, G, act):
    """d/dt sum(y(x + t v) * dy) by central differences of the kernel's own forward, the
    sums in 64 bits.  With h = 2^-6 the cubic term is h^2 of the derivative's scale and the
    rounding of y (2^-22 of it) divides by 2h: together below 2e-3 of |v||dx| in norm."""
    import ugpg
    x, w, b, dy = make(shape, G, dev, torch.float32, act, seed=5)
    g = torch.Generator(device=dev).manual_seed(9)
    v = torch.randn(shape, generator=g, device=dev)
    xr = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(ugpg.group_norm_act(xr, G, w, b, 1e-5, act), (xr,), dy)
    if act == "relu":  # stay on one side of every corner
        h = 2.0 ** -12
    else:
        h = 2.0 ** -6
    f = lambda t: (ugpg.group_norm_act(x + t * v, G, w, b, 1e-5, act).double() * dy.double()).sum()
    num = (f(h) - f(-h)) / (2 * h)
    want = (dx.double() * v.double()).sum()
    size = (dx.double().norm() * v.double().norm()).item()
    assert abs(num.item() - want.item()) <= 2e-3 * size


def test_misaligned_and_strided_inputs(dev):
    """A view one element into its storage (no vector access), and a permuted view."""
    import ugpg
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, dy = make((2, 20, 21, 64), 8, dev, dtype, "silu", seed=2)
        buf = torch.empty(x.numel() + 1, dtype=dtype, device=dev)
        off = buf[1:].view(x.shape).copy_(x)
        assert off.data_ptr() % 16
        want = ugpg.group_norm_act(x, 8, w, b, 1e-5, "silu")
        half = HALF16 if dtype == torch.bfloat16 else 0.0
        got = ugpg.group_norm_act(off, 8, w, b, 1e-5, "silu")
        near(got, want.double(), 32.0, "misaligned", 2 * half)
        perm = x.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(ugpg.group_norm_act(perm, 8, w, b, 1e-5, "silu"), want)


@pytest.mark.parametrize("shape", [(2, 10, 12, 64), (2, 128, 96, 64)])
def test_bad_values_stay_in_their_group(dev, shape):
    """NaN, infinity and the type's lowest value in one group of one sample leave every other
    group's result bit-identical, forward and backward."""
    import ugpg
    x, w, b, dy = make(shape, 8, dev, torch.float32, "relu", seed=4)

    def both(t):
        t = t.clone().requires_grad_(True)
        y = ugpg.group_norm_act(t, 8, w, b)
        return y.detach(), torch.autograd.grad(y, (t,), dy)[0]
    y0, d0 = both(x)
    for bad in (float("nan"), float("inf"), torch.finfo(torch.float32).min):
        z = x.clone()
        z[1, 3, 4, 9] = bad
        y1, d1 = both(z)
        keep = torch.ones(shape, dtype=torch.bool, device=dev)
        keep[1, ..., 8:16] = False
        assert torch.equal(y0[keep], y1[keep]) and torch.equal(d0[keep], d1[keep])
        if bad != bad:
            assert y1[1, ..., 8:16].isnan().all()


def test_same_bits_every_time_and_inside_bounds(dev):
    """Fixed summation order: repeated calls are bit-identical; outputs and gradients inside
    guard bands are all that is written."""
    from tests._guard import guarded
    from ugpg import ops
    for shape, G in (((2, 9, 7, 60), 12), ((2, 128, 96, 64), 32), ((1, 70, 70, 1030), 5)):
        x, w, b, dy = make(shape, G, dev, torch.float32, "relu", seed=6)
        first = None
        for _ in range(3):
            call = ops.GroupNormCall(x, G, w, b, 1e-5, "relu")
            y, mean, rstd = call.forward(), call.mean, call.rstd
            dx = guarded(shape, dev)
            C = shape[-1]
            dw, db, dxs = (guarded((C,), dev) for _ in range(3))
            ops.group_norm_bwd(call, dy, dx.t, dw.t, db.t, dxs.t)
            for n, t in (("dx", dx), ("dw", dw), ("db", db), ("dxsum", dxs)):
                t.check(n)
            now = [y, mean, rstd, dx.t, dw.t, db.t, dxs.t]
            # the sum of dx per channel, against 64 bits
            s = dx.t.double().reshape(-1, C)
            near(dxs.t, s.sum(0), s.abs().sum(0).max().item() + 1.0, "dxsum")
            if first is not None:
                assert all(torch.equal(a, c) for a, c in zip(first, now))
            first = [t.clone() for t in now]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", [((2, 12, 10, 64), 8), ((2, 128, 96, 64), 32)])
def test_mixed_types_of_the_bf16_arithmetic(dev, shape, G, out):
    """x stored in bf16 with a float32 upstream gradient, as the executor calls it."""
    from ugpg import ops
    x, w, b, _ = make(shape, G, dev, torch.bfloat16, "relu", seed=8)
    g = torch.Generator(device=dev).manual_seed(1)
    dy = torch.randn(shape, generator=g, device=dev)
    call = ops.GroupNormCall(x, G, w, b, 1e-5, "relu")
    call.forward()
    dx = torch.empty(shape, dtype=out, device=dev)
    ops.group_norm_bwd(call, dy, dx)
    _, edx, _, _, r = ref(x, G, w, b, 1e-5, "relu", dy)
    near(dx, edx, 512.0 * r.max().item(), "dx", HALF16 if out == torch.bfloat16 else 0.0)
    if out == torch.float32:  # in place over the upstream gradient
        ops.group_norm_bwd(call, dy, dy)
        assert torch.equal(dy, dx)


def test_module_matches_and_keeps_channels_last(dev):
    import torch.nn as nn
    import ugpg
    m = ugpg.GroupNormAct(4, 24, activation="relu").to(dev)
    plain = nn.GroupNorm(4, 24).to(dev)
    plain.load_state_dict(m.state_dict())
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(3, 24, 11, 13, generator=g, device=dev)
    want = torch.relu(plain.double()(x.double()))
    for t in (x, x.contiguous(memory_format=torch.channels_last)):
        y = m(t)
        assert y.shape == x.shape and y.is_contiguous(memory_format=torch.channels_last)
        near(y, want, 32.0, "module")


def test_other_stream_and_captured_graph(dev):
    """On a side stream, and captured with its backward and replayed with new inputs."""
    import ugpg
    for shape, G in (((2, 12, 10, 64), 8), ((2, 128, 96, 64), 32)):
        x, w, b, dy = make(shape, G, dev, torch.float32, "silu", seed=7)

        def step(t, p, q, d):
            y = ugpg.group_norm_act(t, G, p, q, 1e-5, "silu")
            return (y.detach(), *torch.autograd.grad(y, (t, p, q), d))
        leaf = lambda: [t.clone().requires_grad_(True) for t in (x, w, b)]
        want = [t.clone() for t in step(*leaf(), dy)]
        side = torch.cuda.Stream()
        args = leaf()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(*args, dy)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        args = leaf()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*args, dy)
        for k in range(3):
            with torch.no_grad():
                args[0].copy_(x * (1.0 + 0.25 * k))
            graph.replay()
            torch.cuda.synchronize()
            fresh = [t.detach().clone().requires_grad_(True) for t in args]
            ex = step(*fresh, dy)
            assert all(torch.equal(a, c) for a, c in zip(outs, ex)), k


def test_capture_beside_a_living_eager_graph_is_refused(dev):
    """The leaves' accumulators then belong to the default stream, which a captured backward
    may not touch; without the eager graph, or with it on another stream, capture works."""
    import ugpg
    x, w, b, dy = make((2, 12, 10, 64), 8, dev, torch.float32, "silu")
    leaf = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(ugpg.group_norm_act(leaf[0], 8, *leaf[1:], activation="silu"), leaf, dy)
    for which in range(3):
        alive = leaf[which] * 1.0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="default stream"):
                ugpg.group_norm_act(leaf[0], 8, *leaf[1:], activation="silu")
            still = ugpg.group_norm_act(leaf[0].detach(), 8, *(t.detach() for t in leaf[1:]), activation="silu")
        del alive
        graph.replay()
        assert torch.isfinite(still).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ugpg.group_norm_act(leaf[0], 8, *leaf[1:], activation="silu")
        got = torch.autograd.grad(y, leaf, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("C,G", [(64, 8), (16, 1), (4, 4)])
def test_a_chunk_far_from_the_others(dev, C, G):
    """The first pixels of each group's first channel lie 10^4 away from all other values, which
    are equal: the partials' merge must not lose these others' digits.  An output is
    (x - mean) * rstd; mean and rstd are within a few dozen roundings of themselves (a share's
    sums, each about its own first mean), which against x - mean makes EPS32 of
    |x - mean| * rstd + |mean error| * rstd, mean error <= EPS32 * (|mean - x| + |x|)."""
    import ugpg
    x = torch.full((1, 128, 128, C), 0.5, device=dev)
    x[:, 0, :, ::C // G] = 1.0e4
    y = ugpg.group_norm_act(x, G, activation="none")
    xd = x.double().reshape(1, -1, G, C // G)
    mean = xd.mean((1, 3), keepdim=True)
    rstd = ((xd - mean) ** 2).mean((1, 3), keepdim=True).add(1e-5).rsqrt()
    want = ((xd - mean) * rstd).reshape(x.shape)
    lim = EPS32 * (((xd - mean).abs() + (xd - mean).abs() + xd.abs()) * rstd).reshape(x.shape)
    err = (y.double() - want).abs()
    assert (err <= lim).all(), (err / lim).max().item()


def test_differentiable_once(dev):
    """Second derivatives are refused, not silently left out; create_graph alone is fine."""
    import ugpg
    x, w, b, dy = make((2, 6, 5, 24), 4, dev, torch.float32, "silu")
    leaf = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(ugpg.group_norm_act(leaf[0], 4, *leaf[1:], activation="silu"), leaf, dy)
    got = torch.autograd.grad(ugpg.group_norm_act(leaf[0], 4, *leaf[1:], activation="silu"), leaf, dy,
                              create_graph=True)
    assert all(torch.equal(a, c.detach()) for a, c in zip(want, got))
    with pytest.raises(RuntimeError, match="only once"):
        (got[0].sum() + leaf[0].sum()).backward()


def test_offsets_past_32_bits(dev):
    """A bf16 activation of more than 2^32 bytes' worth of elements: the last sample's result
    equals the same sample normalised alone."""
    import ugpg
    B, H, W, C = 9, 512, 1024, 512  # 2.4e9 values: element offsets pass 2^31
    x = torch.empty((B, H, W, C), dtype=torch.bfloat16, device=dev).normal_()
    y = ugpg.group_norm_act(x, 32, activation="relu")
    one = ugpg.group_norm_act(x[B - 1:].clone(), 32, activation="relu")
    d = (y[B - 1].float() - one[0].float()).abs().max().item()
    # other chunks, another summation order: the results differ by float32 roundings, at
    # most one bf16 step (2^-7) of a value of at most 8
    assert d <= 8 * 2.0 ** -7
    assert (y[B - 1].float() != 0).any()
