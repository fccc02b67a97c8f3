"""The bounds of tests/_norm_bounds.py on the CPU: a float32 evaluation of the formula stays within
them, and a result without one of its parts does not."""
import pytest
import torch

from tests import _norm_bounds as nb


def plain32(x, G, w, b, act, dy):
    """The formula in float32 torch operations."""
    B, C = x.shape[0], x.shape[-1]
    xg = x.float().reshape(B, -1, G, C // G)
    wg, bg, d = w.view(1, 1, G, -1), b.view(1, 1, G, -1), dy.float().view(xg.shape)
    c = xg - xg.mean((1, 3), keepdim=True)
    rstd = 1.0 / (c.square().mean((1, 3), keepdim=True) + 1e-5).sqrt()
    xh = c * rstd
    p = xh * wg + bg
    s = torch.sigmoid(p)
    y = {"relu": torch.relu(p), "silu": p * s, "none": p}[act]
    dp = d * {"relu": (p > 0).float(), "silu": s * (1 + p * (1 - s)), "none": torch.ones_like(p)}[act]
    g = dp * wg
    dx = rstd * (g - g.mean((1, 3), keepdim=True) - xh * (g * xh).mean((1, 3), keepdim=True))
    return {"y": y.reshape(x.shape), "dx": dx.reshape(x.shape), "dw": (dp * xh).sum((0, 1)).view(-1),
            "db": dp.sum((0, 1)).view(-1)}


@pytest.mark.parametrize("act", ["relu", "silu", "none"])
@pytest.mark.parametrize("shape,G,D,form", nb.SHAPES)
def test_bounds_hold_and_see_what_is_left_out(shape, G, D, form, act):
    x, w, b, dy = nb.make(shape, G, "cpu", torch.float32, act)
    want = nb.oracle(x, G, w, b, 1e-5, act, dy, D)
    for name, got in plain32(x, G, w, b, act, dy).items():
        assert nb.worst(got, *want[name]) <= 1.0, name
    half = 2.0 ** -8  # the widest comparison: a bfloat16 result
    for part, names in (("s1", ("dx",)), ("s2", ("dx",)), ("pixel", ("dw", "db"))):
        wrong = nb.oracle(x, G, w, b, 1e-5, act, dy, D, without=part)
        for name in names:
            assert nb.worst(wrong[name][0], *want[name], half if name == "dx" else 0.0) > 2.0, (part, name)
