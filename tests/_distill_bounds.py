"""The distillation loss in 64 bits, with bounds for a row whose student is near its teacher.

A row's k + 1 terms are fp64 and its rest's sum of exponentials S is float32, off by r S with
|r| <= REL = 2^-15 (512 roundings of 2^-24: at most 128 additions deep, exponents of at most 126).
The KL's derivative by log S is p_rest - q_rest and its second at most 1/4, so
    |d KL| <= REL |p_rest - q_rest| + REL^2 + 2^-19 KL
(the last: the temperature, rounded to float32 once for all parts, moves the KL by 2^-24 times its
logarithmic derivative, at most 32 KL for exponents up to 16).  The gradient's parts likewise:
    kept   p_j - q_j:              REL p_rest p_j + 2^-19 |p_j - q_j|
    others (p_rest - q_rest) r_v:  REL r_v (p_rest (1 - p_rest) + |p_rest - q_rest|)
and half a step of the stored type.

Class maps take the k + 1 exponentials in float32 too: an exponent x = (t - M) c carries three
roundings, so a probability p = 2^-x is off by 3 ln 2 |x| half steps and 2 of its own; the sum of
p |x| over a row is its entropy, at most log2(17) = 4.1 with 16 entries: 9 + 2 half steps a side,
and 8 for the rest's sum of at most 64 terms and the common factor, make less than 32 of 2^-24 of a
unit of KL: MAP = 2^-19."""
import math

import torch

REL, MAP, KLREL = 2.0 ** -15, 2.0 ** -19, 2.0 ** -19
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def record(teacher, k, T):
    """values, indices, rest of (..., V) logits."""
    v, i = torch.sort(teacher.double(), dim=-1, descending=True, stable=True)
    rest = T * torch.logsumexp(v[..., k:] / T, -1)
    return v[..., :k].to(teacher.dtype), i[..., :k].contiguous(), rest.float()


def oracle(z, v, i, r, T):
    """(R, V) rows -> KL, its bound, the gradient of sum T^2 KL, its bound."""
    z = z.double()
    lq = torch.log_softmax(torch.cat([v.double(), r.double()[:, None]], 1) / T, 1)
    kept = torch.zeros_like(z, dtype=torch.bool).scatter_(1, i, True)
    zr = T * torch.logsumexp(z.masked_fill(kept, -math.inf) / T, 1, keepdim=True)
    lp = torch.log_softmax(torch.cat([z.gather(1, i), zr], 1) / T, 1)
    p, q = lp.exp(), lq.exp()
    kl = (q * (lq - lp)).sum(1)
    pr, qr = p[:, -1:], q[:, -1:]
    gap = (pr - qr).abs()
    klim = REL * gap[:, 0] + REL ** 2 + KLREL * kl + 1e-13
    share = ((z - zr) / T).exp().masked_fill(kept, 0.0)  # r_v
    dz = T * ((pr - qr) * share).scatter_add(1, i, (p - q)[:, :-1])
    dlim = T * (REL * share * (pr * (1 - pr) + gap)).scatter_add(
        1, i, REL * pr * p[:, :-1] + KLREL * (p - q)[:, :-1].abs())
    return kl, klim, dz, dlim + 1e-37
