"""Group norm's results element by element within bounds made of their own terms
(tests/_norm_bounds.py), and its gradient against differences of its own forward along directions
in which it is large or has to vanish."""
import pytest
import torch

from tests import _norm_bounds as nb

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


@pytest.mark.parametrize("act", ["relu", "silu", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G,D,form", nb.SHAPES)
def test_every_element(dev, shape, G, D, form, dtype, act):
    import ugpg
    x, w, b, dy = nb.make(shape, G, dev, dtype, act)
    want = nb.oracle(x, G, w, b, 1e-5, act, dy, D)
    xr, wr, br = (t.clone().requires_grad_(True) for t in (x, w, b))
    y = ugpg.group_norm_act(xr, G, wr, br, 1e-5, act)
    dx, dw, db = torch.autograd.grad(y, (xr, wr, br), dy)
    for name, got in (("y", y.detach()), ("dx", dx), ("dw", dw), ("db", db)):
        assert nb.worst(got, *want[name], HALF[got.dtype]) <= 1.0, name


@pytest.mark.parametrize("act", ["relu", "silu", "none"])
@pytest.mark.parametrize("shape,G,D,form", nb.SHAPES)
def test_executor_call(dev, shape, G, D, form, act):
    """x in bf16 with a float32 upstream gradient and result, and the bias gradient of the
    convolution in front, the sum of dx per channel.  It comes from the channel's totals: beside the
    elements' bounds, two sums of at most 64 roundings, of |w dp| and |xh s2|; an element's bound
    holds the group's mean of the same, and w varies by 1.5 about its mean: 3 times the bounds'
    sum covers all of it."""
    from ugpg import ops
    x, w, b, _ = nb.make(shape, G, dev, torch.bfloat16, act)
    dy = nb.make(shape, G, dev, torch.float32, act)[3]
    want = nb.oracle(x, G, w, b, 1e-5, act, dy, D)
    call = ops.GroupNormCall(x, G, w, b, 1e-5, act)
    call.forward()
    dx = torch.empty_like(dy)
    dw, db, dsum = (torch.empty_like(w) for _ in range(3))
    ops.group_norm_bwd(call, dy, dx, dw, db, dsum)
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        assert nb.worst(got, *want[name]) <= 1.0, name
    flat = lambda t: t.reshape(-1, shape[-1]).sum(0)
    value, limit = want["dx"]
    assert nb.worst(dsum, flat(value), 3.0 * flat(limit)) <= 1.0


@pytest.mark.parametrize("shape,G,D", [((2, 8, 6, 48), 4, 160), ((2, 128, 96, 64), 8, 64)])
@pytest.mark.parametrize("act", ["relu", "silu", "none"])
def test_gradient_against_differences_along_itself(dev, shape, G, D, act):
    """Along u = dx / max|dx| the derivative is |dx|^2 / max|dx|, the largest there is; along a
    constant of each group it has to vanish.  The quotient's own error at this step comes from
    the 64-bit definition, the forward's from its bound over the step."""
    import ugpg
    x, w, b, dy = nb.make(shape, G, dev, torch.float32, act, seed=5)
    want = nb.oracle(x, G, w, b, 1e-5, act, dy, D)
    xr = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(ugpg.group_norm_act(xr, G, w, b, 1e-5, act), (xr,), dy)
    g = torch.Generator(device=dev).manual_seed(6)
    level = torch.randn(shape[0], *[1] * (len(shape) - 2), G, 1, generator=g, device=dev)
    level = level.expand(*shape[:-1], G, shape[-1] // G).reshape(shape)
    h = 2.0 ** -6
    f = lambda t: (ugpg.group_norm_act(t, G, w, b, 1e-5, act).double() * dy.double()).sum().item()
    f64 = lambda t: (nb.oracle(t, G, w, b, 1e-5, act, dy, D)["y"][0] * dy.double()).sum().item()
    for u, large in ((dx / dx.abs().max(), True), (level / level.abs().max(), False)):
        up, down = x + h * u, x - h * u
        u = (up.double() - down.double()) / (2 * h)  # (as the float32 points have it)
        quotient = (f(up) - f(down)) / (2 * h)
        along = (dx.double() * u).sum().item()
        true = (want["dx"][0] * u).sum().item()
        lim = ((dy.double().abs() * want["y"][1]).sum().item() / h
               + abs((f64(up) - f64(down)) / (2 * h) - true) + (want["dx"][1] * u.abs()).sum().item())
        assert abs(quotient - along) <= lim, (quotient, along, lim)
        if large:  # the comparison means something: the bound is a small part of what is compared
            assert lim <= 0.1 * along


@pytest.mark.parametrize("shape,G", [((2, 12, 10, 64), 8), ((2, 128, 96, 64), 32)])
def test_any_subset_of_inputs_gets_its_gradient(dev, shape, G):
    """Weight and bias absent, constant or learned, in every combination."""
    import ugpg
    x, w, b, dy = nb.make(shape, G, dev, torch.float32, "silu", seed=3)
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    for wk in ("none", "constant", "learned"):
        for bk in ("none", "constant", "learned"):
            for xk in ("constant", "learned"):
                xr, wr, br = x.clone(), w.clone(), b.clone()
                leaf = {n: t.requires_grad_(True) for n, t, k in (("dx", xr, xk), ("dw", wr, wk), ("db", br, bk))
                        if k == "learned"}
                y = ugpg.group_norm_act(xr, G, None if wk == "none" else wr, None if bk == "none" else br, 1e-5, "silu")
                want = nb.oracle(x, G, one if wk == "none" else w, zero if bk == "none" else b, 1e-5, "silu", dy, 160)
                assert nb.worst(y.detach(), *want["y"]) <= 1.0
                assert y.requires_grad == bool(leaf)
                if leaf:
                    for name, got in zip(leaf, torch.autograd.grad(y, list(leaf.values()), dy)):
                        assert nb.worst(got, *want[name]) <= 1.0, (wk, bk, xk, name)
