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


def test_captured_backward_into_a_living_eager_graph_is_refused(dev):
    """The leaf lies behind a view, a copy or a cast, so the node itself has no edge to it: the
    backward is refused before it reaches the default stream.  A pass that does not go there, or
    runs without the eager graph, is captured."""
    import ugpg
    torch.manual_seed(4)
    m = ugpg.GroupNormAct(4, 24).to(dev)
    x = torch.randn(2, 24, 6, 5, device=dev, requires_grad=True)
    dy = torch.randn(2, 24, 6, 5, device=dev)
    z = torch.randn(30, 7, device=dev, requires_grad=True)
    top = ugpg.teacher_top_logits(torch.randn(30, 7, device=dev), 3, 2.0)

    def norm(*inputs):
        return torch.autograd.grad(m(x), inputs, dy)

    def loss(*inputs):
        return torch.autograd.grad(ugpg.distillation_loss(z * 2.0, top, 2.0), inputs)
    want = norm(x, m.weight, m.bias) + loss(z)
    for step, leaf in ((norm, x), (loss, z)):
        alive = leaf * 1.0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            still = dy * 2.0
            with pytest.raises(RuntimeError, match="default stream"):
                step(leaf)
            if step is norm:  # the parameters' gradients do not go there
                params = step(m.weight, m.bias)
        del alive
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(still, dy * 2.0)
        if step is norm:
            assert torch.equal(params[0], want[1]) and torch.equal(params[1], want[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = norm(x, m.weight, m.bias) + loss(z)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
