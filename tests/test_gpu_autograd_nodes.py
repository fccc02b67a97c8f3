"""The compiled autograd nodes through the public calls: what they refuse, and which inputs get
a gradient."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu


def test_tangents_are_refused(dev):
    """Forward mode, with and without a reverse graph, and through the module."""
    import ugpg
    x = torch.randn(2, 6, 5, 24, device=dev)
    z = torch.randn(30, 7, device=dev)
    top = ugpg.teacher_top_logits(torch.randn(30, 7, device=dev), 3, 2.0)
    m = ugpg.GroupNormAct(4, 24).to(dev)
    calls = [lambda t: ugpg.group_norm_act(t, 4), lambda t: m(t.movedim(-1, 1))]
    for mode in (torch.enable_grad, torch.no_grad):
        with fwad.dual_level(), mode():
            for call in calls:
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(fwad.make_dual(x, torch.ones_like(x)))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ugpg.distillation_loss(fwad.make_dual(z, torch.ones_like(z)), top, 2.0)
            for call in calls:  # without a tangent the same level changes nothing
                assert torch.isfinite(call(x)).all()
    with pytest.raises(RuntimeError):
        torch.func.jvp(calls[0], (x,), (torch.ones_like(x),))
