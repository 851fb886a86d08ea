"""What the training-step operators are measured on: attention over packed causal sequences, the top-k router with
its balance loss, and the AdamW step over many tensors.

Sizes follow the decoder of the benchmark (hidden 768, 8 query heads over 4 key / value heads, 8 layers, vocabulary
6400, 8 experts, top 2, 8 x 2048 tokens a step) and go out from there to both sides.  ``run`` computes an operator in
elementary torch operations in 32 bits, or, with ``own`` set, through this repository's entry points; ``exact`` gives
the same outputs from the definitions in 64 bits."""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256  # values that share one scale of an 8-bit state
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.95, 1e-8, 0.1


def _package():
    """The package's modules are imported as ``model.*`` from its own folder."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minimind-mhc_b200")
    if at not in sys.path:
        sys.path.insert(0, at)


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a user's short question read before the first answer token: only the latency of the call counts
        {"name": "attn_short", "op": "attn", "dtype": "bf16", "batch": 1, "tokens": 77, "ragged": False, "heads": 8,
         "kv_heads": 4, "dim": 96, "grad": False, "fused": False, "spread": 0},
        # the decoder's training step: 8 rows of 2048 tokens, forward and backward of one layer's attention
        {"name": "attn_train", "op": "attn", "dtype": "bf16", "batch": 8, "tokens": 16384, "ragged": False,
         "heads": 8, "kv_heads": 4, "dim": 96, "grad": True, "fused": False, "spread": 0},
        # fine-tuning on conversations of very different lengths packed into one row, q / k / v slices of one
        # projection's output
        {"name": "attn_packed", "op": "attn", "dtype": "bf16", "batch": 13, "tokens": 8191, "ragged": True,
         "heads": 8, "kv_heads": 2, "dim": 64, "grad": True, "fused": True, "spread": 3},
        # one long document read for evaluation
        {"name": "attn_long", "op": "attn", "dtype": "bf16", "batch": 1, "tokens": 16384, "ragged": False,
         "heads": 8, "kv_heads": 4, "dim": 128, "grad": False, "fused": False, "spread": 0},
        # a training step in full precision, the small model with 8 heads of 64
        {"name": "attn_fp32", "op": "attn", "dtype": "fp32", "batch": 2, "tokens": 1024, "ragged": False, "heads": 8,
         "kv_heads": 8, "dim": 64, "grad": True, "fused": False, "spread": 0},
        # the router of a small batch: latency
        {"name": "router_small", "op": "router", "dtype": "fp32", "tokens": 61, "experts": 8, "k": 2},
        # the router of the decoder's training step
        {"name": "router_train", "op": "router", "dtype": "bf16", "tokens": 16384, "experts": 8, "k": 2},
        # many fine-grained experts over the largest token count of the layer benchmark
        {"name": "router_wide", "op": "router", "dtype": "bf16", "tokens": 262144, "experts": 64, "k": 6},
        # only the connections of one decoder layer are trained (14 small fp32 tensors), gradients clipped
        {"name": "adamw_small", "op": "adamw", "model": "mhc", "layers": 1, "hidden": 768, "vocab": 0,
         "param": "fp32", "bits": 32, "clip": 1.0},
        # the dense decoder under autocast: fp32 parameters and states, gradients clipped to norm 1
        {"name": "adamw_dense", "op": "adamw", "model": "dense", "layers": 8, "hidden": 768, "vocab": 6400,
         "param": "fp32", "bits": 32, "clip": 1.0},
        # the mixture-of-experts decoder of the training benchmark: bf16 matrices, fp32 connections
        {"name": "adamw_moe", "op": "adamw", "model": "moe", "layers": 8, "hidden": 768, "vocab": 6400,
         "param": "bf16", "bits": 32, "clip": 0.0},
        # the same with fp32 parameters and the two moments held in 8 bits
        {"name": "adamw_moe_8bit", "op": "adamw", "model": "moe", "layers": 8, "hidden": 768, "vocab": 6400,
         "param": "fp32", "bits": 8, "clip": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attn", "attn", "router", "adamw"))
    if op == "attn":
        dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32"))
        tokens = _log(rng, 1, 16384 if dtype == "bf16" else 2048)
        batch = min(tokens, _log(rng, 1, 64))
        kv_heads = rng.choice((1, 2, 4, 8))
        return {"op": op, "dtype": dtype, "batch": batch, "tokens": tokens, "ragged": True,
                "heads": 8 if kv_heads > 1 else rng.choice((4, 5, 8)), "kv_heads": kv_heads,
                "dim": rng.choice((32, 64, 80, 96, 128)), "grad": tokens <= 8192 and rng.random() < 0.6,
                "fused": rng.random() < 0.5, "spread": rng.randrange(1, 1 << 20)}
    if op == "router":
        experts = rng.choice((4, 8, 16, 24, 60, 64, 128))
        return {"op": op, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                "tokens": _log(rng, 1, 262144 * 64 // max(64, experts)), "experts": experts,
                "k": rng.randint(1, min(8, experts - 1))}
    model, bits = rng.choice(("mhc", "dense", "moe")), rng.choice((32, 8))
    return {"op": op, "model": model, "layers": rng.randint(1, 8 if model != "moe" else 6),
            "hidden": rng.choice((256, 320, 512, 640, 768)), "vocab": 0 if model == "mhc" else _log(rng, 501, 6400),
            "param": rng.choice(("fp32", "bf16", "fp16")), "bits": bits,
            "clip": rng.choice((0.0, 1.0)) if bits == 32 else 0.0}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths: equal ones, or from one token up to many, drawn from the case's own `spread`."""
    b, t = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [t // b] * b
    rng = random.Random(case["spread"])
    cuts = sorted(rng.sample(range(1, t), b - 1)) if b > 1 else []
    return [hi - lo for lo, hi in zip([0] + cuts, cuts + [t])]


def _shapes(case):
    """The parameters' shapes of the decoder: ([matrices and norms], [the connections' fp32 parameters])."""
    h, layers, n = case["hidden"], case["layers"], 4
    body, conn = [], []
    for _ in range(layers):
        for _ in range(2):
            conn += [(n * h, 2 * n + n * n), (1,), (n,), (1,), (n,), (1,), (n, n)]
        if case["model"] != "mhc":
            body += [(h, h), (h // 2, h), (h // 2, h), (h, h), (h // 8,), (h // 8,), (h,), (h,)]
            inter = 2048 * h // 768
            experts = 8 if case["model"] == "moe" else 1
            body += [(8, h)] if experts > 1 else []
            body += [(inter, h), (h, inter), (inter, h)] * experts
    if case["vocab"]:
        body += [(case["vocab"], h), (h,)]
    return body, conn


def _group(shapes, dtype, bits, gen):
    """Tensors of one dtype as views of flat buffers, each begun at a multiple of BLOCK values, with their gradients
    and moments."""
    dev = "cuda"
    sizes = [math.prod(s) for s in shapes]
    at, total = [], 0
    for s in sizes:
        at.append(total)
        total += -(-s // BLOCK) * BLOCK
    used = torch.zeros(total, device=dev)
    for o, s in zip(at, sizes):
        used[o:o + s] = 1

    def noise(scale):
        return torch.randn(total, device=dev, generator=gen).mul_(scale).mul_(used)

    p, g = noise(0.02).to(dtype), noise(1e-3).to(dtype)
    m, v = noise(3e-4), noise(1e-3).square_().add_(1e-8).mul_(used)
    cut = lambda t: [t[o:o + s].view(shape) for o, s, shape in zip(at, sizes, shapes)]  # noqa: E731
    group = {"p": p, "g": g, "params": cut(p), "grads": cut(g)}
    if bits == 32:
        return group | {"m": m, "v": v, "ms": cut(m), "vs": cut(v)}
    mc, msc = _pack_m(m)
    vc, vsc = _pack_v(v)
    scales = lambda t: [t[o // BLOCK:(o + s + BLOCK - 1) // BLOCK] for o, s in zip(at, sizes)]  # noqa: E731
    return group | {"m": mc, "m_scale": msc, "v": vc, "v_scale": vsc, "ms": list(zip(cut(mc), scales(msc))),
                    "vs": list(zip(cut(vc), scales(vsc)))}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    if case["op"] == "attn":
        dt = DTYPES[case["dtype"]]
        t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        lengths = _lengths(case)
        # what q_norm, k_norm and the value projection leave: unit-scale rows
        if case["fused"]:
            qkv = randn(t, h + 2 * hk, d).to(dt)
            q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        else:
            q, k, v = (randn(t, heads, d).to(dt) for heads in (h, hk, hk))
        cu = torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32)
        if case["grad"]:
            q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        return {"case": case, "q": q, "k": k, "v": v, "cu": cu, "longest": max(lengths),
                "d_out": randn(t, h, d).to(dt) if case["grad"] else None}
    if case["op"] == "router":
        t, e = case["tokens"], case["experts"]
        # router logits of a trained gate: spread over the experts, some of them preferred
        logits = (randn(t, e) + 0.5 * randn(1, e)).to(DTYPES[case["dtype"]]).requires_grad_(True)
        return {"case": case, "logits": logits, "d_weights": randn(t, case["k"]) * 1e-2,
                "d_loss": torch.ones((), device=dev)}
    body, conn = _shapes(case)
    groups = [_group(s, dt, case["bits"], gen)
              for s, dt in ((body, DTYPES[case["param"]]), (conn, torch.float32)) if s]
    lists = {k: [x for g in groups for x in g[k]] for k in ("params", "grads", "ms", "vs")}
    return {"case": case, "groups": groups, "step": 1000, **lists}


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _attention(s):
    """Softmax attention over each packed sequence, causal, the sequences padded to the longest."""
    case = s["case"]
    t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    scale = d ** -0.5
    cu, n = s["cu"].long(), s["longest"]
    pos = torch.arange(n, device=cu.device)
    here = pos[None, :] < (cu[1:] - cu[:-1])[:, None]                  # (B, L)
    at = (cu[:-1, None] + pos[None, :]).clamp(max=t - 1)

    def pad(x, heads):  # (T, heads, D) -> (B, Hkv, heads / Hkv, L, D)
        x = x.detach().float()[at] * here[:, :, None, None]
        return x.view(x.shape[0], n, hk, heads // hk, d).permute(0, 2, 3, 1, 4)

    def unpad(x, heads):
        return x.permute(0, 3, 1, 2, 4).reshape(-1, n, heads, d)[here].to(s["q"].dtype)

    q, k, v = pad(s["q"], h), pad(s["k"], hk), pad(s["v"], hk)
    seen = pos[None, :] <= pos[:, None]
    x = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = p @ v
    if not case["grad"]:
        return {"out": unpad(o, h)}
    do = pad(s["d_out"], h)
    dv = (p.transpose(-1, -2) @ do).sum(2, keepdim=True)
    dp = do @ v.transpose(-1, -2)
    ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return {"out": unpad(o, h), "dq": unpad(ds @ k, h),
            "dk": unpad((ds.transpose(-1, -2) @ q).sum(2, keepdim=True), hk), "dv": unpad(dv, hk)}


COEF = 5e-4  # the decoder's coefficient of the balance loss


def _router(s):
    """Softmax over the experts, the k largest logits of a token (ties: the lowest index), weights that sum to one,
    the experts' counts and coef * E * sum_e (count_e / T) * mean_t p[t, e], and the gradient of the logits."""
    case = s["case"]
    t, e, k = case["tokens"], case["experts"], case["k"]
    z = s["logits"].detach().float()
    ex = (z - z.amax(-1, keepdim=True)).exp()
    p = ex / ex.sum(-1, keepdim=True)
    bits = (z + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * e + torch.arange(e - 1, -1, -1, device=z.device)
    idx = order.topk(k, dim=-1).indices
    top = p.gather(1, idx)
    total = top.sum(-1, keepdim=True) + 1e-20
    w = top / total
    counts = torch.bincount(idx.flatten(), minlength=e)
    load = counts.float() / t
    loss = (load * p.mean(0)).sum() * (e * COEF)
    dw = s["d_weights"]
    dtop = (dw - (dw * w).sum(-1, keepdim=True)) / total
    dp = (load * (s["d_loss"] * (e * COEF / t))).expand(t, e).scatter_add(1, idx, dtop)
    dz = p * (dp - (p * dp).sum(-1, keepdim=True))
    return {"weights": w, "experts": idx, "counts": counts, "loss": loss, "d_logits": dz.to(s["logits"].dtype)}


def _pack_m(m):
    """Signed moments in 8 bits: a block's scale is its largest magnitude, a code the rounded root of the fraction."""
    b = m.view(-1, BLOCK)
    scale = b.abs().amax(1)
    part = b.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    return ((part.sqrt() * 127.0).round() * b.sign()).to(torch.int8).view(-1), scale


def _unpack_m(codes, scale):
    c = codes.view(-1, BLOCK).float()
    return (c * c.abs() * scale[:, None] * (1.0 / 16129.0)).view(-1)


def _pack_v(v):
    """Squares in 8 bits: codes are fourth roots, and what is above zero stays above zero."""
    b = v.view(-1, BLOCK)
    scale = b.amax(1)
    part = b / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    code = (part.sqrt().sqrt() * 255.0).round()
    return torch.where(b > 0, code.clamp(min=1.0), code).to(torch.uint8).view(-1), scale


def _unpack_v(codes, scale):
    c = codes.view(-1, BLOCK).float()
    return (c * c * scale[:, None] * (1.0 / 65025.0) * (c * c) * (1.0 / 65025.0)).view(-1)


def _adamw_group(g, bits, step, clip):
    grad = g["g"].float()
    if clip is not None:
        grad = grad * clip
    m, v = (g["m"], g["v"]) if bits == 32 else (_unpack_m(g["m"], g["m_scale"]), _unpack_v(g["v"], g["v_scale"]))
    m = m * BETA1 + grad * (1 - BETA1)
    v = v * BETA2 + grad * (1 - BETA2) * grad
    denom = v.sqrt() * (1.0 / math.sqrt(1 - BETA2 ** step)) + EPS
    p = g["p"].float() * (1 - LR * DECAY) - m / denom * (LR / (1 - BETA1 ** step))
    g["p"].copy_(p)
    if bits == 32:
        g["m"].copy_(m)
        g["v"].copy_(v)
        return g["p"], g["m"], g["v"]
    for name, (codes, scale) in (("m", _pack_m(m)), ("v", _pack_v(v))):
        g[name].copy_(codes)
        g[name + "_scale"].copy_(scale)
    return g["p"], _unpack_m(g["m"], g["m_scale"]), _unpack_v(g["v"], g["v_scale"])


def _adamw(s):
    """Decoupled weight decay and the step of Adam, in place, on gradients scaled to a norm of at most `clip`."""
    case = s["case"]
    s["step"] += 1
    clip = None
    if case["clip"]:
        norm = sum(g["g"].float().square().sum() for g in s["groups"]).sqrt()
        clip = (case["clip"] / (norm + 1e-6)).clamp(max=1.0)
    return [_adamw_group(g, case["bits"], s["step"], clip) for g in s["groups"]]


# ---------------------------------------------------------------------------
# The repository's entry points
# ---------------------------------------------------------------------------

def _own(s):
    _package()
    case = s["case"]
    if case["op"] == "attn":
        from model.mhc_attention import packed_attention
        q, k, v = s["q"], s["k"], s["v"]
        if case["ragged"]:
            out = packed_attention(q, k, v, s["cu"])
        else:
            rows = (case["batch"], case["tokens"] // case["batch"])
            out = packed_attention(q.unflatten(0, rows), k.unflatten(0, rows), v.unflatten(0, rows)).flatten(0, 1)
        if not case["grad"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["d_out"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if case["op"] == "router":
        from model.mhc_router import route_topk
        w, idx, counts, loss = route_topk(s["logits"], case["k"], aux_coef=COEF)
        dz, = torch.autograd.grad((w, loss), (s["logits"],), (s["d_weights"], s["d_loss"]))
        return {"weights": w.detach(), "experts": idx, "counts": counts, "loss": loss.detach(), "d_logits": dz}
    from model import mhc_adamw
    s["step"] += 1
    common = dict(step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                  max_grad_norm=case["clip"] or None)
    if case["bits"] == 32:
        mhc_adamw.adamw_step(s["params"], s["grads"], s["ms"], s["vs"], **common)
        return [(g["p"], g["m"], g["v"]) for g in s["groups"]]
    mhc_adamw.adamw_step_8bit(s["params"], s["grads"], s["ms"], s["vs"], **common)
    return [(g["p"], mhc_adamw.unpack_moment(g["m"], g["m_scale"]), mhc_adamw.unpack_moment(g["v"], g["v_scale"]))
            for g in s["groups"]]


def run(state):
    if own:
        return _own(state)
    return {"attn": _attention, "router": _router, "adamw": _adamw}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "attn":
        size = 4 if case["dtype"] == "fp32" else 2
        t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        pairs = h * sum(n * (n + 1) // 2 for n in _lengths(case))
        # forward: q, k, v read, out written; the gradients' pass adds d_out read and dq, dk, dv written
        nbytes = size * t * d * (2 * h + 2 * hk) + (size * t * d * (2 * h + 2 * hk) if case["grad"] else 0)
        # two products of 2 D operations for every visible pair, five more for the gradients (the scores again,
        # d_out v^T, and one each for dq, dk, dv)
        return {"bytes": nbytes, "flops": 2 * d * pairs * (2 + (5 if case["grad"] else 0))}
    if case["op"] == "router":
        size = 4 if case["dtype"] == "fp32" else 2
        t, e, k = case["tokens"], case["experts"], case["k"]
        return {"bytes": 2 * size * t * e + t * k * (4 + 8 + 4) + 8 * e, "flops": t * e * 10}
    nbytes, values = 0, 0
    for shapes, size in zip(_shapes(case), ((4 if case["param"] == "fp32" else 2), 4)):
        n = sum(math.prod(x) for x in shapes)
        # parameter and gradient read, parameter written; the moments read and written
        nbytes += n * 3 * size + n * (16 if case["bits"] == 32 else 4)
        # 8-bit moments: their scales, and the values they stand for, which run() returns
        nbytes += 0 if case["bits"] == 32 else n * 8 + 16 * sum(-(-math.prod(x) // BLOCK) for x in shapes)
        values += n
    return {"bytes": nbytes, "flops": values * 14}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_attention(s):
    """One sequence and one key / value head at a time; the gradients are autograd's."""
    case = s["case"]
    grad, dim = case["grad"], case["dim"]
    group = case["heads"] // case["kv_heads"]
    full = [s[x].detach().double() for x in ("q", "k", "v")]
    out = {"out": torch.zeros_like(full[0])}
    if grad:
        out |= {n: torch.zeros_like(x) for n, x in zip(("dq", "dk", "dv"), full)}
        do = s["d_out"].double()
    ends = s["cu"].tolist()
    for lo, hi in zip(ends[:-1], ends[1:]):
        for j in range(case["kv_heads"]):
            heads = slice(j * group, (j + 1) * group)
            k, v = full[1][lo:hi, j], full[2][lo:hi, j]
            step = (hi - lo) if grad else 2048
            for a in range(lo, hi, step):
                b = min(hi, a + step)
                q, kk, vv = full[0][a:b, heads], k[:b - lo], v[:b - lo]
                if grad:
                    q, kk, vv = (x.detach().requires_grad_(True) for x in (q, kk, vv))
                logits = torch.einsum("ihd,jd->hij", q, kk) / math.sqrt(dim)
                later = torch.arange(b - lo, device=k.device)[None] > torch.arange(a - lo, b - lo, device=k.device)[:, None]
                o = torch.einsum("hij,jd->ihd", torch.softmax(logits.masked_fill(later, -math.inf), -1), vv)
                out["out"][a:b, heads] = o.detach()
                if grad:
                    g = torch.autograd.grad(o, (q, kk, vv), do[a:b, heads])
                    out["dq"][a:b, heads], out["dk"][lo:hi, j], out["dv"][lo:hi, j] = g
    return out


def _exact_router(s):
    case = s["case"]
    z = s["logits"].detach().double().requires_grad_(True)
    p = torch.softmax(z, -1)
    # a stable sort keeps the lower index first among equals
    idx = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[:, :case["k"]]
    top = p.gather(1, idx)
    w = top / (top.sum(-1, keepdim=True) + 1e-20)
    chosen = torch.zeros_like(z).detach().scatter_(1, idx, 1.0)
    loss = COEF * case["experts"] * (chosen.mean(0) * p.mean(0)).sum()
    dz, = torch.autograd.grad((w, loss), (z,), (s["d_weights"].double(), s["d_loss"].double()))
    return {"weights": w.detach(), "experts": idx, "counts": chosen.sum(0).long(), "loss": loss.detach(),
            "d_logits": dz}


def _exact_adamw(s):
    case = s["case"]
    step = s["step"] + 1
    factor = 1.0
    if case["clip"]:
        norm = torch.stack([g["g"].double().pow(2).sum() for g in s["groups"]]).sum().sqrt()
        factor = torch.clamp(case["clip"] / (norm + 1e-6), max=1.0)
    got = []
    for g in s["groups"]:
        grad, m, v = g["g"].double() * factor, g["m"].double(), g["v"].double()
        if case["bits"] == 8:
            by = lambda name: g[name + "_scale"].double().repeat_interleave(BLOCK)  # noqa: E731
            m, v = (m / 127).square() * m.sign() * by("m"), (v / 255).pow(4) * by("v")
        m.mul_(BETA1).add_(grad, alpha=1 - BETA1)
        v.mul_(BETA2).add_(grad.square_(), alpha=1 - BETA2)
        del grad
        change = (m / (1 - BETA1 ** step)).div_((v / (1 - BETA2 ** step)).sqrt_().add_(EPS))
        p = g["p"].double().mul_(1 - LR * DECAY).sub_(change, alpha=LR)
        del change
        if case["bits"] == 8:
            top = m.abs().view(-1, BLOCK).amax(1, keepdim=True)
            code = torch.round(127 * (m.abs().view(-1, BLOCK) / top.clamp(min=1e-300)).sqrt())
            m = ((code / 127).square() * top).view(-1) * m.sign()
            top = v.view(-1, BLOCK).amax(1, keepdim=True)
            code = torch.round(255 * (v.view(-1, BLOCK) / top.clamp(min=1e-300)).pow(0.25))
            code = torch.where(v.view(-1, BLOCK) > 0, code.clamp(min=1), code)
            v = ((code / 255).pow(4) * top).view(-1)
        got.append((p, m, v))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attention, "router": _exact_router, "adamw": _exact_adamw}[case["op"]](s)
