"""The bounds of tests/_distill_bounds.py on the CPU: float32 terms of a row break them, a float32
sum of the rest does not."""
import math

import pytest
import torch

from tests import _distill_bounds as db


def half_precise(z, v, i, r, T, terms):
    """The KL with the rest's exponentials summed in float32 and the k + 1 terms in `terms`."""
    kept = torch.zeros_like(z, dtype=torch.bool).scatter_(1, i, True)
    o = z.masked_fill(kept, -math.inf)
    m = o.amax(1, keepdim=True)
    s = ((o - m) / T).exp().sum(1, keepdim=True)
    zz = torch.cat([z.gather(1, i).to(terms) / T, m.to(terms) / T + s.to(terms).log()], 1)
    tt = torch.cat([v.to(terms), r.to(terms)[:, None]], 1) / T
    lq, lp = torch.log_softmax(tt, 1), torch.log_softmax(zz, 1)
    return (lq.exp() * (lq - lp)).sum(1)


@pytest.mark.parametrize("noise", [0.0, 1e-3])
@pytest.mark.parametrize("V,k", [(50, 5), (3000, 40)])
def test_bounds_tell_float32_terms(V, k, noise):
    g = torch.Generator().manual_seed(V)
    t = 2.0 * torch.randn(200, V, generator=g)
    z = t + noise * torch.randn(200, V, generator=g)
    v, i, r = db.record(t, k, 2.0)
    kl, lim, _, _ = db.oracle(z, v, i, r, 2.0)
    assert ((half_precise(z, v, i, r, 2.0, torch.float64) - kl).abs() <= lim).all()
    off = (half_precise(z, v, i, r, 2.0, torch.float32).double() - kl).abs()
    assert (off > lim).float().mean() > 0.1  # most rows at noise 0
