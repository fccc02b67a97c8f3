"""Networks with norm="group": the executor's forward, gradients and training steps against
the same network written in torch on the CPU, under both arithmetics, in graphs, and the cell
classifier taught by its previous stage (group norm, top logits and distillation together)."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from oracle import detgen as G

pytestmark = pytest.mark.gpu


def plain_double_conv(dc, x):
    for c, n in ((dc.conv_op[0], dc.conv_op[1]), (dc.conv_op[3], dc.conv_op[4])):
        x = F.relu(F.group_norm(F.conv2d(x, c.weight, c.bias, padding=1), n.num_groups, n.weight, n.bias, n.eps))
    return x


def plain_forward(m, x):
    """PGUNet{1..4} with group norm, in torch ops on the module's own parameters."""
    from ugpg.unet import _LAYOUT
    _, enc, dec, heads = _LAYOUT[m.STAGE]
    feats = [plain_double_conv(m.inc.conv, x)]
    for name, _, _ in enc:
        feats.append(plain_double_conv(getattr(m, name).double_conv, F.max_pool2d(feats[-1], 2)))
    low, outs = feats[-1], []
    for i, (name, _, _) in enumerate(dec):
        skip = feats[len(feats) - 2 - i]
        up = F.interpolate(low, scale_factor=2, mode="bilinear", align_corners=True)
        low = plain_double_conv(getattr(m, name).double_conv, torch.cat([skip, up], 1))
        h = getattr(m, heads[i]).conv
        outs.append(F.conv2d(low, h.weight, h.bias))
    hw = outs[-1].shape[-2:]
    return sum(F.interpolate(o, size=hw, mode="bilinear", align_corners=True) if o.shape[-2:] != hw else o
               for o in outs)


def grads_of(m, x, t, dtype, seed=None, rel=0.0):
    m = copy.deepcopy(m).cpu().to(dtype)
    if seed is not None:
        with torch.no_grad():
            for k, p in m.named_parameters():
                p.mul_(1 + rel * G.randn(seed, tuple(p.shape), k).to(dtype))
    y = plain_forward(m, x.to(dtype))
    F.binary_cross_entropy_with_logits(y, t.to(dtype)).backward()
    return y.detach(), {k: p.grad for k, p in m.named_parameters()}


@pytest.mark.parametrize("stage,res,groups", [(1, 32, 32), (2, 64, 8), (4, 64, 16)])
def test_network_matches_torch(dev, stage, res, groups):
    """Gradients against 64 bits within 3 times what one-ulp-sized changes of the weights do to
    torch's own float32 run (near-ties of ReLU and max-pool flip), the rule of the BatchNorm
    networks; logits within 1e-3."""
    import ugpg
    torch.manual_seed(stage)
    m = getattr(ugpg, f"PGUNet{stage}")(3, 1, norm="group", groups=groups)
    assert not list(m.buffers())
    with torch.no_grad():
        for k, p in m.named_parameters():
            if p.dim() == 1:
                p.add_(0.1 * G.randn(9, tuple(p.shape), k))
    x = G.randn(31, (2, 3, res, res), "x")
    t = G.bernoulli(32, (2, 1, res, res), 0.5, "t")
    y64, g64 = grads_of(m, x, t, torch.float64)
    y32, g32 = grads_of(m, x, t, torch.float32)
    floor = {k: (g32[k].double() - g64[k]).abs().max().item() for k in g64}
    for seed, rel in ((7, 1e-7), (8, 1e-7), (9, 1e-6), (10, 5e-6)):
        _, gp = grads_of(m, x, t, torch.float32, seed, rel)
        for k in floor:
            floor[k] = max(floor[k], (gp[k].double() - g64[k]).abs().max().item())
    g = m.to(dev)
    y = g(x.to(dev))
    F.binary_cross_entropy_with_logits(y, t.to(dev)).backward()
    assert (y.detach().cpu().double() - y64).abs().max().item() <= 1e-3
    for k, p in g.named_parameters():
        err = (p.grad.cpu().double() - g64[k]).abs().max().item()
        bound = 3 * floor[k] + 1e-6 * g64[k].abs().max().item()
        assert err <= bound, (k, err, bound)
    g.eval()  # no running statistics: the same function, to the bit
    with torch.no_grad():
        assert torch.equal(g(x.to(dev)), y.detach())


def test_sample_does_not_depend_on_the_batch(dev):
    """What the norm is for: an image's logits do not depend on the others (to the summation
    orders' roundings: kernels choose tiles by the batch)."""
    import ugpg
    torch.manual_seed(0)
    m = ugpg.PGUNet2(3, 1, norm="group").to(dev)
    x = G.randn(5, (5, 3, 64, 64), "x").to(dev)
    with torch.no_grad():
        assert (m(x)[3:4] - m(x[3:4])).abs().max().item() <= 1e-4


def test_blocks_standalone(dev):
    import ugpg
    torch.manual_seed(3)
    for blk, args in ((ugpg.DoubleConv(64, 64, norm="group", groups=8), [(2, 64, 32, 32)]),
                      (ugpg.Down(64, 128, norm="group"), [(2, 64, 32, 32)]),
                      (ugpg.Up(128, 64, norm="group"), [(2, 64, 16, 16), (2, 64, 32, 32)])):
        blk = blk.to(dev)
        xs = [G.randn(7 + i, s, "x").to(dev).requires_grad_(True) for i, s in enumerate(args)]
        out = blk(*xs)
        c64 = copy.deepcopy(blk).cpu().double()
        x64 = [x.detach().cpu().double().requires_grad_(True) for x in xs]
        if len(xs) == 2:
            up = F.interpolate(x64[0], scale_factor=2, mode="bilinear", align_corners=True)
            ref = plain_double_conv(c64.double_conv, torch.cat([x64[1], up], 1))
        elif isinstance(blk, ugpg.Down):
            ref = plain_double_conv(c64.double_conv, F.max_pool2d(x64[0], 2))
        else:
            ref = plain_double_conv(c64, x64[0])
        assert (out.detach().cpu().double() - ref.detach()).abs().max().item() <= 1e-4
        w = G.randn(11, tuple(out.shape), "w")
        (out * w.to(dev)).sum().backward()
        (ref * w.double()).sum().backward()
        for a, b in zip(xs, x64):  # norm-wise: single ReLU near-ties may flip
            assert (a.grad.cpu().double() - b.grad).norm().item() <= 1e-3 * b.grad.norm().item()


def test_bf16_arithmetic(dev):
    """bf16 storage of the conv outputs: logits within the bf16 arithmetic's spread of the
    float32 ones (2^-8 a rounding, some thirty roundings deep), gradients along them."""
    import ugpg
    from ugpg import ops
    torch.manual_seed(1)
    m = ugpg.PGUNet4(3, 1, norm="group").to(dev)
    x = G.randn(41, (2, 3, 64, 64), "x").to(dev)
    t = G.bernoulli(42, (2, 1, 64, 64), 0.5, "t").to(dev)

    def run(math):
        old = ops.conv_math()
        ops.set_conv_math(math)
        try:
            m.zero_grad()
            y = m(x)
            F.binary_cross_entropy_with_logits(y, t).backward()
            return y.detach().clone(), torch.cat([p.grad.reshape(-1) for p in m.parameters()]).double()
        finally:
            ops.set_conv_math(old)
    y32, g32 = run("x6")
    y16, g16 = run("bf16")
    assert (y16 - y32).norm().item() <= 30 * 2.0 ** -8 * y32.norm().item()
    cos = (g16 @ g32 / (g16.norm() * g32.norm())).item()
    assert cos >= 1 - 30 * 2.0 ** -8, cos
    assert not torch.equal(y16, y32)


def test_trainer_step_and_graphs(dev):
    """Two uncertainty-guided steps of stage 3 with group norm: the captured step equals the
    eager one bit for bit, and the loss is finite."""
    import ugpg

    def make():
        torch.manual_seed(99)
        tr = ugpg.UncertaintyGuidedProgressiveTrainer(3, 1, device=dev, norm="group", norm_groups=16)
        tr.stage_configs[2]["resolution"], tr.stage_configs[3]["resolution"] = 32, 64
        tr.current_stage, tr.current_model = 3, tr.models[3]
        tr.setup_optimizer(3)
        tr.current_model.train()
        tr.models[2].eval()
        return tr
    A, B = make(), make()
    B.enable_graphs()
    g = torch.Generator().manual_seed(3)
    for k in range(5):
        x = torch.randn(2, 3, 64, 64, generator=g).to(dev)
        t = (torch.rand(2, 1, 64, 64, generator=g) < 0.5).float().to(dev)
        a, b = A.train_step(x, t, 3).tolist(), B.train_step(x, t, 3).tolist()
        assert a == b and a[0] == a[0], (k, a, b)
    assert B.last_step_graph is not None and B.last_step_graph.replays >= 3
    for p, q in zip(A.current_model.parameters(), B.current_model.parameters()):
        assert torch.equal(p, q)


def herlev_config(dev, **kw):
    return dict(device=dev, epochs_per_stage=1, num_classes=7, stage4_resolution=64, stages=[1, 2], **kw)


def test_classifier_taught_by_its_previous_stage(dev):
    """HerlevTrainer with group norm and distill_weight: its loss is the uncertainty-guided one
    plus the distillation written out from the previous stage's logits, and so is its gradient."""
    import ugpg  # noqa: F401
    from ugpg.herlev import HerlevTrainer
    torch.manual_seed(5)
    tr = HerlevTrainer(herlev_config(dev, norm="group", norm_groups=16, distill_weight=0.7, distill_top=3,
                                     distill_temperature=2.0))
    plain = tr.distillation
    model, prev = tr.models[2], tr.models[1]
    assert isinstance(model.unet.inc.conv.conv_op[1], nn.GroupNorm)
    for mod in model.modules():
        if isinstance(mod, nn.Dropout):
            mod.p = 0.0
    model.train()
    x = G.randn(61, (6, 3, 64, 64), "x").to(dev)
    y = torch.tensor([0, 1, 2, 3, 4, 6], device=dev)

    def step():
        model.zero_grad()
        output, final, out = tr._forward_device(x, y, 2)
        final.backward()
        return output.detach(), final.detach(), out, [p.grad.clone() for p in model.parameters() if p.grad is not None]
    out1, f1, m1, g1 = step()
    tr.distillation = None
    out0, f0, m0, g0 = step()
    tr.distillation = plain
    assert torch.equal(out0, out1)
    # the distillation term in 64 bits
    with torch.no_grad():
        from ugpg import ops
        t = prev(ops.resize_nchw(x, 32, 32, ops.RESIZE_BILINEAR)).double()
    z = out0.double().requires_grad_(True)
    v, i = t.sort(1, descending=True)
    rest = 2.0 * torch.logsumexp(v[:, 3:] / 2.0, 1, keepdim=True)
    q = torch.softmax(torch.cat([v[:, :3], rest], 1) / 2.0, 1)
    lp = torch.log_softmax(z / 2.0, 1).gather(1, i)
    logp = torch.cat([lp[:, :3], torch.logsumexp(lp[:, 3:], 1, keepdim=True)], 1)
    d = 0.7 * 4.0 * (q * (q.log() - logp)).sum(1).mean()
    (dz,) = torch.autograd.grad(d, (z,))
    assert abs((f1 - f0).item() - d.item()) <= 1e-5 * (1 + abs(f0.item()))
    assert m1[0].item() == pytest.approx(f1.item(), rel=1e-6) and torch.equal(m0[1:], m1[1:])
    # its gradient through the network: the difference of the two backward passes equals the
    # backward of dz alone (float32 rounding of gradients of size |g0| + |g1|)
    model.zero_grad()
    output = model(x)
    output.backward(dz.float())
    for a, b, p in zip(g1, g0, [p for p in model.parameters() if p.grad is not None]):
        lim = 1e-4 * (a.abs().max() + b.abs().max() + p.grad.abs().max()).item()
        assert (a - b - p.grad).abs().max().item() <= lim
    # and a whole training step, and an evaluation
    tr.setup_optimizer_scheduler(2)
    before = [p.detach().clone() for p in model.parameters()]
    tr.train_step(x, y, 2)
    assert any(not torch.equal(a, b) for a, b in zip(before, model.parameters()))
    model.eval()
    with torch.no_grad():
        tr._forward_device(x, y, 2)


def test_binary_classifier_is_taught_too(dev):
    from ugpg.herlev import HerlevTrainer
    torch.manual_seed(6)
    cfg = herlev_config(dev, distill_weight=1.0, distill_top=3)
    cfg["num_classes"] = 2
    tr = HerlevTrainer(cfg)
    assert tr.distillation.k == 2
    x, y = G.randn(62, (2, 3, 64, 64), "x").to(dev), torch.tensor([0, 1], device=dev)
    tr.models[2].train()
    tr.setup_optimizer_scheduler(2)
    m = tr.train_step(x, y, 2)
    assert m[0].isfinite()


def test_progressive_driver_and_evaluation(dev, tmp_path):
    """train_progressive over the four stages with group norm: weights carry over, and the
    checkpoint loads for evaluation with its norm and groups."""
    import ugpg
    torch.manual_seed(8)
    tr = ugpg.UncertaintyGuidedProgressiveTrainer(3, 1, device=dev, norm="group", norm_groups=8)
    for s in tr.stage_configs:
        tr.stage_configs[s]["epochs_per_stage"] = 1
    g = torch.Generator().manual_seed(1)
    batch = [(torch.rand(2, 3, 64, 64, generator=g), (torch.rand(2, 1, 64, 64, generator=g) < 0.5).float())]
    tr.train_progressive(batch, batch, save_dir=str(tmp_path))
    files = sorted(tmp_path.glob("ug_pgunet_stage4_best.pth"))
    assert files, list(tmp_path.iterdir())
    te = ugpg.MoNuSegTester(str(files[0]), device=dev)
    assert te.model.inc.conv.conv_op[1].num_groups == 8
    masks, conf = te.predict(torch.rand(1, 3, 256, 256, generator=g))
    assert masks.shape == (1, 1, 256, 256)
