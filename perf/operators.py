"""The operators a stage trains with when its batch is small and the previous stage teaches
it, each as a user calls it and in its plain form:

  group_norm_act      group normalisation with an activation on channels-last images, with
                      its backward pass (what replaces BatchNorm + ReLU in a DoubleConv when
                      a GPU holds too few images for batch statistics)
  teacher_top_logits  the k largest logits of every row of a teacher's output, and the one
                      logit that stands for all the others
  distillation_loss   KL divergence from that record to a student's logits, with its gradient

Rows are the rows of an (N, V) matrix, or the pixels of an (N, V, H, W) class map.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "ug-pg-unet_amd")
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5


def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _ugpg():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import ugpg
    return ugpg


# ---------------------------------------------------------------- cases
def _gn(name, B, H, W, C, G, act, dtype, train):
    return dict(name=name, op="group_norm_act", B=B, H=H, W=W, C=C, G=G, act=act, dtype=dtype,
                train=train)


def _ds(name, N, V, k, dtype, H=0, W=0, T=2.0, rest=True, weight=True, train=True):
    return dict(name=name, op="distillation_loss", N=N, V=V, H=H, W=W, k=k, T=T, rest=rest,
                weight=weight, dtype=dtype, train=train)


def _tk(name, N, V, k, dtype, H=0, W=0, T=1.0):
    return dict(name=name, op="teacher_top_logits", N=N, V=V, H=H, W=W, k=k, T=T, dtype=dtype)


def listed():
    return [
        # the bottleneck of one 256^2 image (down4's output), evaluation: latency counts
        _gn("gn_fwd_bottleneck_one_image", 1, 16, 16, 512, 32, "relu", "f32", False),
        # down1's width at half resolution, 16 images in bf16 storage, evaluation
        _gn("gn_fwd_bf16_down1", 16, 128, 128, 128, 32, "relu", "bf16", False),
        # the first block at full resolution, 16 images: the largest activation of a step
        _gn("gn_train_inc_bs16", 16, 256, 256, 64, 32, "relu", "f32", True),
        # odd image sizes, 5 channels a group, a smooth activation
        _gn("gn_train_bf16_odd", 6, 75, 53, 60, 12, "silu", "bf16", True),
        # the 7-class cell classifier at batch 16, taught by the previous stage
        _ds("distill_classifier", 16, 7, 3, "f32"),
        # a wide output layer in bf16, thousands of rows: bandwidth
        _ds("distill_wide_bf16", 4096, 32768, 64, "bf16"),
        # rows of odd length (no row but the first is aligned), a record without its rest
        _ds("distill_odd_f32", 517, 50003, 20, "f32", T=1.0, rest=False),
        # dense multi-class maps at full resolution, weighted by an uncertainty map
        _ds("distill_maps", 16, 8, 3, "f32", H=256, W=256),
        # three very long rows, validation only: few rows must still fill the card
        _ds("distill_eval_few_rows", 3, 131071, 256, "bf16", T=1.5, train=False),
        # recording a teacher's outputs for later epochs
        _tk("top_wide_bf16", 2048, 131072, 128, "bf16", T=2.0),
        # one row: what a single request records
        _tk("top_one_row", 1, 65537, 50, "f32"),
        # the teacher's class maps, three classes kept of eight
        _tk("top_maps", 16, 8, 3, "f32", H=256, W=256, T=2.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["group_norm_act", "distillation_loss", "teacher_top_logits"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "group_norm_act":
        G = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 32, 64])
        C = G * _log_int(rng, 1, max(1, min(64, 1024 // G)))
        H, W = _log_int(rng, 4, 256), _log_int(rng, 4, 256)
        B = max(1, min(_log_int(rng, 1, 32), (16 * 256 * 256 * 64) // (H * W * C)))
        return dict(op=op, B=B, H=H, W=W, C=C, G=G, act=rng.choice(["relu", "silu", "none"]),
                    dtype=dtype, train=rng.random() < 0.6)
    maps = rng.random() < 0.25
    limit = 4096 * 32768 if op == "distillation_loss" else 2048 * 131072
    if maps:
        V, H, W = _log_int(rng, 2, 64), _log_int(rng, 8, 256), _log_int(rng, 8, 256)
        N = max(1, min(_log_int(rng, 1, 16), (16 * 8 * 256 * 256) // (V * H * W)))
        k = rng.randint(1, min(V, 8))
    else:
        V, H, W = _log_int(rng, 3, 131072), 0, 0
        N = max(1, min(_log_int(rng, 1, 8192), limit // V))
        k = _log_int(rng, 1, min(V, 256))
    T = rng.choice([0.5, 1.0, 1.5, 2.0, 4.0])
    case = dict(op=op, N=N, V=V, H=H, W=W, k=k, T=T, dtype=dtype)
    if op == "distillation_loss":
        case.update(rest=rng.random() < 0.7, weight=rng.random() < 0.7, train=rng.random() < 0.7)
    return case


# ---------------------------------------------------------------- inputs
def _shape(case):
    sp = (case["H"], case["W"]) if case["H"] else ()
    return (case["N"], case["V"], *sp)


def _teacher(case, g):
    """Logits with a broad body and a few confident classes a row; a long row's last five
    places are unused ones, masked to -inf, as a padded output layer's are."""
    z = torch.randn(_shape(case), generator=g, device=_dev()) * 2.0
    if case["V"] > 100:
        hot = torch.randint(0, case["V"] - 5, (case["N"], 8), generator=g, device=_dev())
        z.scatter_add_(1, hot, 8.0 * torch.rand(hot.shape, generator=g, device=_dev()))
        z[:, -5:] = -math.inf
    return z


def _ordered(z):
    """int64 keys that sort as (value, then the lower index first) does; z fp32, no NaN."""
    b = (z + 0.0).view(torch.int32)
    b = (b ^ ((b >> 31) & 0x7FFFFFFF)).long()
    last = z.shape[-1] - 1
    return (b << 32) + (last - torch.arange(z.shape[-1], device=z.device))


def _plain_top(z, k, T):
    """z (..., V) -> values, indices, rest, in fp32."""
    z = z.float()
    idx = _ordered(z).topk(k, dim=-1).indices
    val = z.gather(-1, idx)
    body = z.scatter(-1, idx, -math.inf)
    m = body.amax(-1, keepdim=True)
    safe = torch.where(m == -math.inf, torch.zeros_like(m), m)
    rest = m + T * ((body - safe) / T).exp().sum(-1, keepdim=True).log()
    rest = torch.where(m == -math.inf, m, rest)
    return val, idx, rest.squeeze(-1)


def _off_corner(x, G, w, b):
    """Move values whose normalised value lies within 1e-3 of the activation's corner off it:
    the ReLU's derivative jumps there, and the side would be rounding's choice."""
    B, H, W, C = x.shape
    xd = x.double().view(B, H * W, G, C // G)
    mean = xd.mean((1, 3), keepdim=True)
    std = (xd - mean).square().mean((1, 3), keepdim=True).add(_EPS).sqrt()
    gap = w.double().view(1, 1, G, -1)
    pre = ((xd - mean) / std * gap + b.double().view(1, 1, G, -1)).view(x.shape)
    step = (0.05 * std / gap).expand_as(xd).reshape(x.shape)
    near = pre.abs() < 1e-3
    return torch.where(near, (x.double() + torch.where(pre < 0, -step, step)), x.double()).to(x.dtype)


def prepare(case, seed):
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DT[case["dtype"]]
    rn = lambda *s: torch.randn(s, generator=g, device=dev)
    st = dict(case=case)
    if case["op"] == "group_norm_act":
        B, H, W, C, G = (case[n] for n in ("B", "H", "W", "C", "G"))
        # a conv's output: channels of different offset and spread
        x = (rn(B, H, W, C) * (0.5 + torch.rand(C, generator=g, device=dev)) + 0.5 * rn(C)).to(dt)
        w = 0.5 + torch.rand(C, generator=g, device=dev)
        b = 0.3 * rn(C)
        if case["act"] == "relu" and case["train"]:
            x = _off_corner(x, G, w, b)
        st.update(x=x, w=w, b=b)
        if case["train"]:
            st["dy"] = (rn(B, H, W, C) / math.sqrt(H * W)).to(dt)
            for n in ("x", "w", "b"):
                st[n].requires_grad_(True)
        return st
    teacher = _teacher(case, g).to(dt)
    if case["op"] == "teacher_top_logits":
        st["logits"] = teacher
        return st
    val, idx, rest = _plain_top(teacher.movedim(1, -1), case["k"], case["T"])
    if case["k"] > 1:  # a third of the rows kept fewer: their last entries are absent
        short = torch.rand(rest.shape, generator=g, device=dev) < 1.0 / 3.0
        val[..., -1] = torch.where(short, torch.full_like(rest, math.nan), val[..., -1])
        idx[..., -1] = torch.where(short, torch.full_like(idx[..., -1], -1), idx[..., -1])
    noise = torch.randn(teacher.shape, generator=g, device=dev)
    student = (teacher.float() + noise).to(dt)
    wt = None
    if case["weight"]:  # 1 + an uncertainty in [0, 1]; one row in sixteen is padding
        wt = 1.0 + torch.rand(rest.shape, generator=g, device=dev)
        wt = torch.where(torch.rand(rest.shape, generator=g, device=dev) < 1 / 16, 0.0, wt)
    st.update(logits=student.requires_grad_(case["train"]),
              values=val.movedim(-1, 1).to(dt).contiguous(),
              indices=idx.movedim(-1, 1).contiguous(),
              rest=rest.contiguous() if case["rest"] else None, weight=wt)
    return st


# ---------------------------------------------------------------- plain forms
def _act(p, act):
    if act == "relu":
        return p * (p > 0)
    if act == "silu":
        return p / (1.0 + (-p).exp())
    return p


def _act_grad(p, act):
    if act == "relu":
        return (p > 0).float()
    if act == "silu":
        s = 1.0 / (1.0 + (-p).exp())
        return s * (1.0 + p * (1.0 - s))
    return torch.ones_like(p)


def _plain_gn(st):
    c = st["case"]
    B, HW, G, D = c["B"], c["H"] * c["W"], c["G"], c["C"] // c["G"]
    x = st["x"].detach()
    w, b = (st[n].detach().view(1, 1, G, D) for n in ("w", "b"))
    xf = x.float().view(B, HW, G, D)
    d = xf - xf.mean((1, 3), keepdim=True)
    rstd = 1.0 / (d.square().mean((1, 3), keepdim=True) + _EPS).sqrt()
    xh = d * rstd
    p = xh * w + b
    y = _act(p, c["act"]).to(x.dtype).view(x.shape)
    if not c["train"]:
        return y
    dp = st["dy"].float().view(xf.shape) * _act_grad(p, c["act"])
    dw, db = (dp * xh).sum((0, 1)).view(-1), dp.sum((0, 1)).view(-1)
    dxh = dp * w
    dx = rstd * (dxh - dxh.mean((1, 3), keepdim=True) - xh * (dxh * xh).mean((1, 3), keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype).view(x.shape), "dw": dw, "db": db}


def _plain_distill(st):
    c = st["case"]
    T, logits = c["T"], st["logits"].detach()
    z = logits.movedim(1, -1).float()
    V = z.shape[-1]
    val, idx = st["values"].movedim(1, -1).float(), st["indices"].movedim(1, -1)
    there = (idx >= 0) & (idx < V)
    ninf = torch.full_like(val, -math.inf)
    t = torch.where(there, val, ninf)
    zi = torch.where(there, z.gather(-1, idx.clamp(0, V - 1)), ninf)
    # absent entries mark nothing: they point one place past the row
    mark = torch.zeros(*z.shape[:-1], V + 1, dtype=torch.bool, device=z.device)
    mark = mark.scatter(-1, torch.where(there, idx, torch.full_like(idx, V)), True)[..., :V]
    body = torch.where(mark, torch.full_like(z, -math.inf), z)
    m = z.amax(-1, keepdim=True)
    e_body = ((body - m) / T).exp()
    # the long sum, and the few terms whose difference the loss is, in 64 bits
    s_body = e_body.sum(-1, keepdim=True, dtype=torch.float64)
    zi, m = zi.double(), m.double()
    e_top = ((zi - m) / T).exp()
    s = s_body + e_top.sum(-1, keepdim=True)
    r = st["rest"]
    r = ninf[..., :1] if r is None else r.unsqueeze(-1)
    tt = torch.cat([t, r], -1).double()
    tm = tt.amax(-1, keepdim=True)
    q = ((tt - tm) / T).exp()
    q = q / q.sum(-1, keepdim=True)
    logp = torch.cat([(zi - m) / T, s_body.log()], -1) - s.log()
    kl = torch.where(q > 0, q * (q.log() - logp), torch.zeros_like(q)).sum(-1)
    wt = st["weight"]
    wt = torch.ones_like(kl) if wt is None else wt
    n = kl.numel()
    loss = (T * T * torch.where(wt != 0, wt * kl, torch.zeros_like(kl)).sum() / n).float()
    if not c["train"]:
        return loss
    coef = (T / n * wt).unsqueeze(-1)
    p_top, q_top = e_top / s, q[..., :-1]
    grow = 1.0 - q[..., -1:] * s / s_body
    dz = torch.where(mark, torch.zeros_like(z), e_body * (coef / s * grow).float())
    part = torch.where(there, coef * (p_top - q_top), torch.zeros_like(q_top)).float()
    dz = dz.scatter_add(-1, idx.clamp(0, V - 1), part)
    return {"loss": loss, "dlogits": dz.movedim(-1, 1).to(logits.dtype).contiguous()}


def _plain_topk(st):
    c, z = st["case"], st["logits"]
    val, idx, rest = _plain_top(z.movedim(1, -1), c["k"], c["T"])
    back = lambda t: t.movedim(-1, 1).contiguous()
    return {"values": back(val).to(z.dtype), "indices": back(idx), "rest": rest}


# ---------------------------------------------------------------- the framework's calls
def _own(st):
    u, c = _ugpg(), st["case"]
    if c["op"] == "group_norm_act":
        y = u.group_norm_act(st["x"], c["G"], st["w"], st["b"], _EPS, c["act"])
        if not c["train"]:
            return y
        dx, dw, db = torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if c["op"] == "teacher_top_logits":
        top = u.teacher_top_logits(st["logits"], c["k"], c["T"])
        return {"values": top.values, "indices": top.indices, "rest": top.rest}
    top = u.TopLogits(st["values"], st["indices"], st["rest"])
    loss = u.distillation_loss(st["logits"], top, c["T"], weight=st["weight"])
    if not c["train"]:
        return loss
    (dz,) = torch.autograd.grad(loss, (st["logits"],))
    return {"loss": loss.detach(), "dlogits": dz}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "group_norm_act":
        return _plain_gn(state)
    return _plain_distill(state) if op == "distillation_loss" else _plain_topk(state)


# ---------------------------------------------------------------- work and 64-bit definitions
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "group_norm_act":
        n = case["B"] * case["H"] * case["W"] * case["C"]
        # x in, y out; training also dy in, dx out
        return {"bytes": n * es * (4 if case["train"] else 2) + 16 * case["C"],
                "flops": n * (24 if case["train"] else 8)}
    rows = case["N"] * max(1, case["H"] * case["W"])
    n, rec = rows * case["V"], rows * (case["k"] * (es + 8) + 4)
    if case["op"] == "teacher_top_logits":
        return {"bytes": n * es + rec, "flops": 4 * n}
    wt = 4 * rows if case["weight"] else 0
    return {"bytes": n * es * (2 if case["train"] else 1) + rec + wt + 4,
            "flops": n * (8 if case["train"] else 4)}


def _exact_gn(st):
    c = st["case"]
    G, act = c["G"], c["act"]
    x, w, b = (st[n].detach().double().requires_grad_(c["train"]) for n in ("x", "w", "b"))
    B, H, W, C = x.shape
    groups = x.reshape(B, H * W, G, C // G).transpose(1, 2).reshape(B, G, -1)
    var, mean = torch.var_mean(groups, dim=2, unbiased=False)
    norm = (groups - mean[..., None]) * torch.rsqrt(var + _EPS)[..., None]
    norm = norm.view(B, G, H * W, C // G).transpose(1, 2).reshape(B, H, W, C)
    pre = norm * w + b
    y = {"relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v), "none": lambda v: v}[act](pre)
    if not c["train"]:
        return y
    dx, dw, db = torch.autograd.grad(y, (x, w, b), st["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _exact_top(case, logits):
    z = logits.double().movedim(1, -1)
    out_v, out_i, out_r = [], [], []
    flat = z.reshape(-1, z.shape[-1])
    step = max(1, (1 << 27) // z.shape[-1])
    for lo in range(0, flat.shape[0], step):
        v, i = torch.sort(flat[lo:lo + step], dim=-1, descending=True, stable=True)
        k = case["k"]
        out_v.append(v[:, :k])
        out_i.append(i[:, :k])
        out_r.append(case["T"] * torch.logsumexp(v[:, k:] / case["T"], -1) if k < v.shape[1]
                     else torch.full_like(v[:, 0], -math.inf))
    lead = z.shape[:-1]
    cat = lambda p: torch.cat(p).view(*lead, -1).movedim(-1, 1).contiguous()
    return {"values": cat(out_v), "indices": cat(out_i), "rest": torch.cat(out_r).view(lead)}


def _exact_distill(st):
    """One extended row per row: the kept classes, then the rest as one class."""
    c = st["case"]
    T = c["T"]
    z = st["logits"].detach().double().movedim(1, -1)
    V = z.shape[-1]
    lead = z.shape[:-1]
    z = z.reshape(-1, V)
    val = st["values"].double().movedim(1, -1).reshape(len(z), -1)
    idx = st["indices"].movedim(1, -1).reshape(len(z), -1)
    there = idx >= 0
    t = val.masked_fill(~there, -math.inf)
    r = st["rest"].double().reshape(-1, 1) if st["rest"] is not None else None
    logq = torch.log_softmax(torch.cat([t, r], 1) / T if r is not None else t / T, 1)
    q = logq.exp()
    wt = (st["weight"].double().reshape(-1) if st["weight"] is not None
          else torch.ones(len(z), dtype=torch.float64, device=z.device))
    coef = wt / len(z)
    logp = torch.log_softmax(z / T, 1)
    kept = torch.zeros_like(z, dtype=torch.bool)
    rows = torch.arange(len(z), device=z.device)[:, None].expand_as(idx)
    kept[rows[there], idx[there]] = True
    logp_top = logp.gather(1, idx.clamp_min(0)).masked_fill(~there, -math.inf)
    logp_rest = torch.logsumexp(logp.masked_fill(kept, -math.inf), 1)
    both = torch.cat([logp_top, logp_rest[:, None]], 1) if r is not None else logp_top
    terms = torch.where(q > 0, q * (logq - both), torch.zeros_like(q))
    loss = T * T * (coef * terms.sum(1)).sum()
    if not c["train"]:
        return loss
    dz = logp.exp()
    if r is not None:
        back = (logp - logp_rest[:, None]).exp().nan_to_num(0.0) * q[:, -1:]
        dz = dz - back.masked_fill(kept, 0.0)
    dz[rows[there], idx[there]] -= q[:, :idx.shape[1]][there]
    dz = dz * (T * coef)[:, None]
    return {"loss": loss, "dlogits": dz.view(*lead, V).movedim(-1, 1).contiguous()}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "group_norm_act":
        return _exact_gn(st)
    if case["op"] == "teacher_top_logits":
        return _exact_top(case, st["logits"].detach())
    return _exact_distill(st)
