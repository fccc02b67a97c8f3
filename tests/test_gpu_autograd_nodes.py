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


def test_recomputed_and_from_two_threads(dev):
    """Under activation checkpointing, and in two host threads on streams of their own, the
    gradients are the plain call's bits."""
    import threading

    import ugpg
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(7)
    top = ugpg.teacher_top_logits(torch.randn(2, 24, 16, 12, device=dev), 3, 2.0)
    x0 = torch.randn(2, 16, 12, 24, device=dev)
    w0, b0 = torch.rand(24, device=dev) + 0.5, torch.randn(24, device=dev)

    def both(x, w, b):
        y = ugpg.group_norm_act(x, 4, w, b, 1e-5, "silu")
        return ugpg.distillation_loss(y.movedim(-1, 1), top, 2.0)

    def grads(run, scale):
        leaf = [t.clone().requires_grad_(True) for t in (x0, w0, b0)]
        loss = run(*leaf)
        return (loss.detach(), *torch.autograd.grad(scale * loss, leaf))
    want = {s: grads(both, s) for s in (1.0, 3.0)}
    for s in want:
        got = grads(lambda *a: checkpoint(both, *a, use_reentrant=False), s)
        assert all(torch.equal(p, q) for p, q in zip(got, want[s]))
    torch.cuda.synchronize()
    wrong = []

    def work(s):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = grads(both, s)
                stream.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want[s])):
                    wrong.append(s)
    threads = [threading.Thread(target=work, args=(s,)) for s in want]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_graphed_callables(dev):
    """Forward and backward captured apart (torch.cuda.make_graphed_callables), replayed with new
    inputs and upstream factors."""
    import ugpg
    torch.manual_seed(8)
    top = ugpg.teacher_top_logits(torch.randn(40, 24, device=dev), 3, 2.0)

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = ugpg.GroupNormAct(4, 24, activation="silu")

        def forward(self, x):
            return ugpg.distillation_loss(self.norm(x), top, 2.0)
    eager = Net().to(dev)
    graphed = Net().to(dev)
    graphed.load_state_dict(eager.state_dict())
    graphed = torch.cuda.make_graphed_callables(graphed, (torch.randn(40, 24, device=dev, requires_grad=True),))
    for k in range(4):
        x = torch.randn(40, 24, device=dev)
        out = []
        for net in (eager, graphed):
            leaf = x.clone().requires_grad_(True)
            loss = net(leaf) * (1.0 if k % 2 else 2.5)
            loss.backward()
            out.append([loss.detach().clone(), leaf.grad.clone(),
                        *(p.grad.clone() for p in net.parameters())])
            net.zero_grad(set_to_none=True)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(*out)), k
