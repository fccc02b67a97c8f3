"""Tangents of forward-mode differentiation are refused, not silently left out (no GPU needed: the
nodes look before they touch any memory).  The record of a teacher is a constant by definition."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


def dual(t):
    return fwad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_group_norm_refuses_tangents(mode, grad):
    from ugpg._nodes import nodes
    x, w, b = torch.randn(2, 5, 8), torch.ones(8), torch.zeros(8)
    for which in range(3):
        with fwad.dual_level(), mode():
            args = [t.clone().requires_grad_(grad) for t in (x, w, b)]
            args[which] = dual(args[which])
            with pytest.raises(NotImplementedError, match="forward-mode"):
                nodes().group_norm_act(*args, 4, 1e-5, 1)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_distillation_refuses_tangents(mode, grad):
    from ugpg._nodes import nodes
    z, v, i = torch.randn(4, 9), torch.randn(4, 3), torch.arange(3).expand(4, 3).contiguous()
    r, w = torch.randn(4), torch.ones(4)
    for which in (0, 1, 3, 4):
        with fwad.dual_level(), mode():
            args = [z.clone().requires_grad_(grad), v, i, r, w]
            args[which] = dual(args[which])
            with pytest.raises(NotImplementedError, match="forward-mode"):
                nodes().distill(*args, 2.0, 1.0, False)
