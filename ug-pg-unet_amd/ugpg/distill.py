"""Distillation from a teacher's top logits: the previous stage as a teacher.

The reference lets the frozen previous stage only weight the loss by its uncertainty
(Herlev/train_herlev.py:216-296, UG_unet.py:61-94).  Here its output can be learned from as
well: ``teacher_top_logits`` records the k largest logits of every row (or pixel) and the one
logit that stands for all the others, ``distillation_loss`` is the KL divergence from that
record to a student's logits, with its gradient.  A record can be kept (it is k values and
indices a row instead of all classes) and read in later epochs.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import ops
from ._nodes import nodes


class TopLogits(NamedTuple):
    """A teacher's record: ``values`` and ``indices`` (N, k, *spatial), ``rest`` (N, *spatial)
    = T * logsumexp(others / T), or None for no mass beyond the record.  An entry whose
    index lies outside the classes (-1) is absent, its value unused."""
    values: torch.Tensor
    indices: torch.Tensor
    rest: Optional[torch.Tensor] = None


def _check_logits(what, logits):
    if logits.dim() < 2:
        raise ValueError(f"{what}: expected (N, classes, *spatial) logits, got {tuple(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{what}: logits must be float32 or bfloat16, got {logits.dtype}")
    if logits.numel() == 0:
        raise ValueError(f"{what}: empty logits {tuple(logits.shape)}")
    if logits.shape[1] > 1 << 30:
        raise ValueError(f"{what}: {logits.shape[1]} classes are too many")
    rows = logits.numel() // logits.shape[1]
    if rows > ops.ROWS_MAX and rows == logits.shape[0]:
        raise ValueError(f"{what}: {rows} rows, at most {ops.ROWS_MAX} rows a call")
    if rows > ops.PIXELS_MAX:
        raise ValueError(f"{what}: {rows} pixels, at most {ops.PIXELS_MAX} pixels a call")


def _check_temperature(what, t):
    if not 1e-30 <= float(t) <= 1e30:
        raise ValueError(f"{what}: temperature must lie in 1e-30..1e30, got {t}")


def _check_device(what, logits):
    if not logits.is_cuda:
        raise RuntimeError("ugpg: tensor is not on a ROCm/HIP device (no CPU fallback)")


def teacher_top_logits(logits, k, temperature=1.0):
    """The ``k`` largest logits of every row of (N, V) -- or of every pixel of (N, V, *spatial)
    -- the larger first and equal ones by the lower index, and the rest's logit at
    ``temperature``.  float32 or bfloat16; 1 <= k <= min(V, 256); at most 2^22 rows, or 2^30 - 64
    pixels.  A constant: no gradient."""
    what = "teacher_top_logits"
    _check_logits(what, logits)
    _check_temperature(what, temperature)
    if not isinstance(k, int) or not 1 <= k <= min(logits.shape[1], ops.TOP_MAX):
        raise ValueError(f"{what}: k must be an int in 1..{min(logits.shape[1], ops.TOP_MAX)}, got {k!r}")
    _check_device(what, logits)
    return TopLogits(*nodes().top_logits(logits, k, temperature))


def distillation_loss(logits, top, temperature=1.0, weight=None, reduction="mean", scale=1.0):
    """scale * T^2 * reduction(weight * KL(teacher || student)) over the rows of ``logits``
    (N, V) or the pixels of (N, V, *spatial), float32 or bfloat16.

    ``top``: a TopLogits (or a tuple like one) recorded at the same temperature; both
    distributions live on its classes and, where it has a ``rest``, all the others as one.
    ``weight``: one float32 factor a row (N, *spatial); a row of weight 0 gives neither loss
    nor gradient, whatever it holds.  ``reduction``: "mean" (over all rows, as the
    uncertainty-weighted loss), "sum" or "none".  Class maps have at most 1024 classes;
    rows and pixels as for teacher_top_logits.
    The gradient goes to ``logits`` alone (once); record and weight are constants."""
    what = "distillation_loss"
    _check_logits(what, logits)
    _check_temperature(what, temperature)
    top = TopLogits(*top)
    values, indices, rest = top
    lead = (logits.shape[0], *logits.shape[2:])
    k = values.shape[1] if values.dim() > 1 else 0
    if values.dim() != logits.dim() or (values.shape[0], *values.shape[2:]) != lead \
            or not 1 <= k <= min(logits.shape[1], ops.TOP_MAX):
        raise ValueError(f"{what}: values {tuple(values.shape)} do not fit logits "
                         f"{tuple(logits.shape)} with 1..{min(logits.shape[1], ops.TOP_MAX)} entries")
    if indices.shape != values.shape:
        raise ValueError(f"{what}: indices {tuple(indices.shape)} vs values {tuple(values.shape)}")
    if values.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{what}: values must be float32 or bfloat16, got {values.dtype}")
    if indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: indices must be int32 or int64, got {indices.dtype}")
    for name, t in (("rest", rest), ("weight", weight)):
        if t is None:
            continue
        if tuple(t.shape) != lead:
            raise ValueError(f"{what}: {name} must have shape {lead}, got {tuple(t.shape)}")
        if t.dtype != torch.float32:
            raise TypeError(f"{what}: {name} must be float32, got {t.dtype}")
    for name, t in (("values", values), ("indices", indices), ("rest", rest), ("weight", weight)):
        if t is None:
            continue
        if t.device != logits.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, logits on {logits.device}")
        if t.requires_grad:
            raise ValueError(f"{what}: {name} is a constant of the loss; detach it")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"{what}: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if not float(scale) == float(scale):
        raise ValueError(f"{what}: scale is not a number")
    spatial = logits.numel() // (lead[0] * logits.shape[1])
    if spatial > 1 and logits.shape[1] > ops.MAP_CLASSES:
        raise ValueError(f"{what}: class maps of {logits.shape[1]} classes (at most {ops.MAP_CLASSES}); "
                         "pass (pixels, classes) rows")
    _check_device(what, logits)
    if reduction == "mean":
        scale = float(scale) / (lead[0] * spatial)
    if not values.is_contiguous():
        values = values.contiguous()
    if not indices.is_contiguous():
        indices = indices.contiguous()
    if rest is not None and not rest.is_contiguous():
        rest = rest.contiguous()
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    return nodes().distill(logits, values, indices, rest, weight, temperature, scale, reduction == "none")


class DistillationLoss:
    """distillation_loss with its settings: call it on a student's logits and the teacher's
    logits (or a TopLogits recorded earlier)."""

    def __init__(self, k, temperature=2.0, scale=1.0, reduction="mean"):
        if not isinstance(k, int) or not 1 <= k <= ops.TOP_MAX:
            raise ValueError(f"DistillationLoss: k must be an int in 1..{ops.TOP_MAX}, got {k!r}")
        _check_temperature("DistillationLoss", temperature)
        self.k, self.temperature, self.scale, self.reduction = k, temperature, scale, reduction

    def __call__(self, logits, teacher, weight=None):
        if isinstance(teacher, torch.Tensor):
            teacher = teacher_top_logits(teacher, min(self.k, teacher.shape[1]), self.temperature)
        return distillation_loss(logits, teacher, self.temperature, weight, self.reduction, self.scale)
