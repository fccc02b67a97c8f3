"""Group norm with an activation in 64 bits, with a bound for every element of a float32
implementation's results, from the terms that are actually there.

e = 2^-24 is half a step.  D counts the roundings along the longest chain of a statistic's sum:
runs of 4 pixels, a tree of up to 9 levels and a handful of chunks, of 4 roundings each (D = 64),
or, where a block holds its group in registers, up to 16 vectors of 8 values one after the other
and then a tree (D = 160).  Each is relative to the mean |x| of the values it covers, so
  |d mean| <= D e mean|x|,   |d rstd| <= D e rstd      (centred squares: nothing cancels)
  |d xh| <= rho (1 + |xh|),  rho = D e (1 + mean|x| rstd)
and from there on by the chain rule, 4 roundings a line; SiLU's derivative is at most 1.1, that
of its derivative at most 0.5, and the exponential's relative error of (2|p| + 4) e reaches the
result as |p| s (1 - s) (2|p| + 4) e <= 2 e.  Sums over a channel or a group: at most 64 roundings
of the sum of the terms' absolute values."""
import torch

E = 2.0 ** -24
SUM = 64


def oracle(x, G, w, b, eps, act, dy, D, without=None):
    """-> {name: (value, bound)} for y, dx, dw, db.  `without` leaves a part out, to show that the
    bounds see it: "s1" / "s2" (a group mean of dx), "pixel" (the last one of dw and db)."""
    B, C = x.shape[0], x.shape[-1]
    xg = x.detach().double().reshape(B, -1, G, C // G)
    wg, bg = (t.detach().double().view(1, 1, G, -1) for t in (w, b))
    dyg = dy.detach().double().view(xg.shape)
    mean = xg.mean((1, 3), keepdim=True)
    rstd = ((xg - mean) ** 2).mean((1, 3), keepdim=True).add(eps).rsqrt()
    xh = (xg - mean) * rstd
    p = xh * wg + bg
    rho = D * E * (1.0 + xg.abs().mean((1, 3), keepdim=True) * rstd)
    exh = rho * (1.0 + xh.abs())
    ep = wg.abs() * exh + 2 * E * (p.abs() + (wg * xh).abs())
    s = torch.sigmoid(p)
    if act == "silu":
        y, d1 = p * s, s * (1.0 + p * (1.0 - s))
        ey, edp = 1.1 * ep + 4 * E * y.abs() + 2 * E, dyg.abs() * (0.5 * ep + 8 * E)
    elif act == "relu":  # (no pre-activation within its error of the corner)
        y, d1 = torch.relu(p), (p > 0).double()
        ey, edp = ep, torch.zeros_like(p)
    else:
        y, d1 = p, torch.ones_like(p)
        ey, edp = ep, torch.zeros_like(p)
    dp = dyg * d1
    gmean = lambda t: t.mean((1, 3), keepdim=True)
    s1, s2 = gmean(wg * dp), gmean(wg * dp * xh)
    es1 = gmean(wg.abs() * edp) + SUM * E * gmean((wg * dp).abs())
    es2 = gmean(wg.abs() * (edp * xh.abs() + dp.abs() * exh)) + SUM * E * gmean((wg * dp * xh).abs())
    dx = rstd * (wg * dp - (0.0 if without == "s1" else s1) - (0.0 if without == "s2" else xh * s2))
    edx = rstd * (wg.abs() * edp + es1 + xh.abs() * es2 + s2.abs() * exh +
                  4 * E * ((wg * dp).abs() + s1.abs() + (xh * s2).abs())) + rho * dx.abs()
    over = lambda t: t.sum((0, 1)).view(-1)
    db, dw = dp.clone(), dp * xh
    if without == "pixel":
        db[-1, -1] = dw[-1, -1] = 0.0
    edb = over(edp) + SUM * E * over(dp.abs())
    edw = over(edp * xh.abs() + dp.abs() * exh) + SUM * E * over((dp * xh).abs())
    flat = lambda t: t.reshape(x.shape)
    return {"y": (flat(y), flat(ey)), "dx": (flat(dx), flat(edx)), "dw": (over(dw), edw), "db": (over(db), edb)}


def worst(got, want, limit, half=0.0):
    """The largest error over its bound; `half`: half a step of the result's own type."""
    return ((got.double() - want).abs() / (limit + half * want.abs() + 1e-300)).max().item()


def make(shape, G, dev, dtype, act, seed=0):
    """x, w, b, and an upstream gradient with a mean and a component along the normalised values,
    so that both group means of dx are of the size of dy."""
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g, device=dev)
    B, C = shape[0], shape[-1]
    x = rn(*shape) + 0.5 * rn(C)
    w = 0.5 + torch.rand(C, generator=g, device=dev)
    b = 0.3 * rn(C)
    x = x.to(dtype)

    def normed(t):
        tg = t.double().reshape(B, -1, G, C // G)
        m = tg.mean((1, 3), keepdim=True)
        std = ((tg - m) ** 2).mean((1, 3), keepdim=True).add(1e-5).sqrt()
        return ((tg - m) / std).reshape(shape), std.expand_as(tg).reshape(shape)
    if act == "relu":  # which side of the corner a value falls on would be rounding's choice
        xh, std = normed(x)
        p = xh * w.double() + b.double()
        x = torch.where(p.abs() < 1e-3, x.double() + torch.where(p < 0, -0.05, 0.05) * std / w.double(),
                        x.double()).to(dtype)
    dy = rn(*shape) + 0.5 + 0.5 * normed(x)[0].float()
    return x, w, b, dy.to(dtype)


# shape, groups, D, form
SHAPES = [
    ((2, 12, 10, 64), 8, 160, "resident"),
    ((4, 16, 16, 512), 32, 160, "resident"),
    ((2, 5, 3, 60), 12, 160, "resident, 5 channels a group"),
    ((2, 64, 64, 256), 8, 160, "resident in bf16"),
    ((2, 128, 96, 64), 32, 64, "two passes"),
    ((1, 200, 211, 7), 7, 64, "two passes, odd channels"),
    ((3, 75, 53, 60), 12, 64, "two passes, ragged"),
    ((1, 130, 128, 320), 4, 64, "two passes, wide groups"),
    ((1, 70, 70, 1030), 5, 64, "two passes, a merge launch"),
]
