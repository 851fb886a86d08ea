"""What the operators of answering are measured on: rotary positions, the paged cache of keys and values with the
attention that reads it, and the verification of drafted tokens.

One step of a decoder that answers with drafted tokens runs them in this order: every sequence brings its last token
and a tree of drafted ones; their queries and keys are rotated, the keys and values appended to the sequence's pages;
attention over the cache lets a drafted token see the context and its own ancestors; the target's probabilities decide
which drafted tokens are kept, and the kept ones' cache rows are moved up.  Training and evaluation use the rotation
alone, with its gradient.

Sizes follow the decoder of the benchmark (8 query heads over 4 key / value heads of 96, theta 1e6, vocabulary 6400,
8 layers, 8 x 2048 tokens a training step) and go out from there to both sides.  ``run`` computes an operator in
elementary torch operations in 32 bits, or, with ``own`` set, through this repository's entry points; ``exact`` gives
the same outputs from the definitions in 64 bits."""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


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
        # the decoder's training step: queries and keys of 8 rows of 2048 tokens, and the gradients of both
        {"name": "rotate_train", "op": "rotate", "dtype": "bf16", "tokens": 16384, "rows": 8, "heads": 8, "kv_heads": 4,
         "dim": 96, "part": 96, "interleaved": False, "factor": 1, "far": 0, "grad": True, "fused": False},
        # a long document read in full precision, positions scaled beyond the trained length, neighbouring elements
        # paired, three quarters of a head rotated, q and k slices of one projection's output
        {"name": "rotate_long", "op": "rotate", "dtype": "fp32", "tokens": 8191, "rows": 0, "heads": 8, "kv_heads": 2,
         "dim": 128, "part": 96, "interleaved": True, "factor": 16, "far": 1000000, "grad": False, "fused": True},
        # one more token for each of 16 sequences: latency
        {"name": "append_step", "op": "append", "dtype": "bf16", "batch": 16, "new": 1, "context": 2048, "heads": 8,
         "kv_heads": 4, "dim": 96, "part": 96, "interleaved": False, "page": 64, "factor": 1, "spread": 0},
        # prompts of different lengths read into an empty cache
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "batch": 24, "new": 1024, "context": 0, "heads": 8,
         "kv_heads": 4, "dim": 96, "part": 96, "interleaved": False, "page": 64, "factor": 1, "spread": 1},
        # the first tokens of an answer to a short question: only the latency of the call counts
        {"name": "attend_one", "op": "attend", "dtype": "bf16", "batch": 1, "new": 1, "tree": False, "context": 200,
         "heads": 8, "kv_heads": 4, "dim": 96, "page": 64, "spread": 2},
        # a server's step without drafts: 64 sequences of very different lengths
        {"name": "attend_step", "op": "attend", "dtype": "bf16", "batch": 64, "new": 1, "tree": False, "context": 8192,
         "heads": 8, "kv_heads": 4, "dim": 96, "page": 64, "spread": 3},
        # 16 sequences with a tree of up to 63 drafted tokens each, four query heads for a key head
        {"name": "attend_trees", "op": "attend", "dtype": "bf16", "batch": 16, "new": 64, "tree": True, "context": 16384,
         "heads": 8, "kv_heads": 2, "dim": 128, "page": 32, "spread": 4},
        # one very long document with a small tree: the keys have to be shared out
        {"name": "attend_long", "op": "attend", "dtype": "bf16", "batch": 1, "new": 16, "tree": True, "context": 131072,
         "heads": 8, "kv_heads": 4, "dim": 128, "page": 16, "spread": 5},
        # five tokens drafted in a row for one sequence, the decoder's vocabulary: latency
        {"name": "verify_chain", "op": "verify", "batch": 1, "new": 6, "tree": False, "vocab": 6400, "draft": True,
         "spread": 6},
        # 32 sequences with trees of up to 31 drafted tokens and a large vocabulary
        {"name": "verify_trees", "op": "verify", "batch": 32, "new": 32, "tree": True, "vocab": 100003, "draft": True,
         "spread": 7},
        # the kept tokens of one sequence in the decoder's 8 layers
        {"name": "keep_one", "op": "keep", "dtype": "bf16", "layers": 8, "batch": 1, "new": 16, "context": 500,
         "kv_heads": 4, "dim": 96, "page": 64, "spread": 8},
        # and of 64 sequences
        {"name": "keep_many", "op": "keep", "dtype": "bf16", "layers": 8, "batch": 64, "new": 48, "context": 700,
         "kv_heads": 4, "dim": 96, "page": 64, "spread": 9},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotate", "rotate", "append", "append", "attend", "attend", "attend", "attend", "verify", "verify",
                     "keep"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    dim = rng.choice((32, 40, 64, 80, 96, 96, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 8) if g * kv_heads <= 16])
    page = rng.choice((8, 16, 17, 32, 64, 100, 128))
    spread = rng.randrange(10, 1 << 20)
    part = rng.choice((dim, dim, dim // 2, 2 * (dim // 6)))
    position = {"part": part, "interleaved": rng.random() < 0.5, "factor": rng.choice((1, 1, 4, 16))}
    if op == "rotate":
        rows = rng.choice((0, 0, 1, 3, 8))
        tokens = _log(rng, 1, 16384 * 96 // max(96, dim) * 12 // max(12, heads + kv_heads))
        return {"op": op, "dtype": dtype, "tokens": -(-tokens // max(1, rows)) * max(1, rows), "rows": rows, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, **position, "far": rng.choice((0, 0, 30000, 1000000)) if rows == 0 else 0,
                "grad": rng.random() < 0.6, "fused": rng.random() < 0.5}
    if op == "append":
        batch = _log(rng, 1, 64)
        return {"op": op, "dtype": dtype, "batch": batch, "new": _log(rng, 1, max(1, 12000 // batch)),
                "context": _log(rng, 1, 2048) - 1, "heads": heads, "kv_heads": kv_heads, "dim": dim, **position, "page": page,
                "spread": spread}
    if op == "attend":
        new = rng.choice((1, 1, _log(rng, 2, 64), _log(rng, 2, 64)))
        tree = new > 1 and rng.random() < 0.7
        if new > 1 and not tree and rng.random() < 0.5:  # a piece of a long prompt
            new = _log(rng, 64, 400)
        batch = _log(rng, 1, max(1, 1500 // new if new > 64 else 64 if new < 8 else 16))
        most = min(131072, 262144 // batch // kv_heads * 2, 12000000 // (batch * new * heads) if dtype != "fp32" else 1500000 // (batch * new * heads))
        return {"op": op, "dtype": dtype, "batch": batch, "new": new, "tree": tree, "context": _log(rng, 1, max(2, most)) - 1,
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "spread": spread}
    if op == "verify":
        batch, new = _log(rng, 1, 32), _log(rng, 1, 32)
        return {"op": op, "batch": batch, "new": new, "tree": rng.random() < 0.7,
                "vocab": _log(rng, 500, min(150000, 64000000 // (batch * new))), "draft": rng.random() < 0.7, "spread": spread}
    return {"op": op, "dtype": dtype, "layers": rng.randint(1, 8), "batch": _log(rng, 1, 48), "new": _log(rng, 2, 48),
            "context": _log(rng, 1, 600) - 1, "kv_heads": rng.choice((1, 2, 4)), "dim": dim, "page": page, "spread": spread}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _steps(case):
    """(context lengths, new tokens, parents within the sequence) of every sequence, from the case's own `spread`: the
    first of several has all that the case allows, the others anything down to an empty cache and one token."""
    rng = random.Random(case["spread"])
    contexts, news, parents = [], [], []
    for b in range(case["batch"]):
        first, most = b == 0, case.get("context", 0)
        contexts.append(most if first else rng.randint(most // 2, most) if rng.random() < 0.5 else _log(rng, 1, most + 1) - 1)
        n = case["new"] if first else _log(rng, max(1, case["new"] // 2), case["new"])
        news.append(n)
        # a tree grows by a child of one of its newest nodes, so that it is deep and wide; without one it is a chain
        parents.append([-1] + [(rng.randrange(max(0, j - 8), j) if case.get("tree") else j - 1) for j in range(1, n)])
    return contexts, news, parents


def _ancestors(parents):
    """For every node the bits of itself and its ancestors, and its depth."""
    bits, depth = [], []
    for j, p in enumerate(parents):
        bits.append((1 << j) | (bits[p] if p >= 0 else 0))
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return bits, depth


def _signed(x):
    return x - (1 << 64) if x >> 63 else x


def _inv_freq(part, theta, factor, original=2048, fast=32.0, slow=1.0):
    """theta^(-2i / part); beyond the trained length the slow ones are divided by the factor, the fast ones left, by a
    ramp between the frequencies that turn `slow` and `fast` times within it."""
    f = theta ** (-torch.arange(0, part, 2, dtype=torch.float64) / part)
    if factor == 1:
        return f, 1.0
    at = lambda turns: part * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), part // 2 - 1)
    ramp = ((torch.arange(part // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f * (1 - ramp + ramp / factor), 0.1 * math.log(factor) + 1.0


def _positions_plan(case, s):
    f, gain = _inv_freq(case["part"], 1e6, case["factor"])
    s["inv_freq"], s["gain"] = f.to("cuda"), gain
    if own:
        _package()
        from model.mhc_rotary import Rotary
        s["rotary"] = Rotary(case["part"], 1e6, interleaved=case["interleaved"], factor=case["factor"],
                             original_length=2048 if case["factor"] != 1 else None)


def _pages(case, contexts, news, gen):
    """A table of pages in random order, wide enough for the longest sequence, and how many pages there are."""
    need = [-(-(c + n) // case["page"]) for c, n in zip(contexts, news)]
    total = sum(need) + 1
    order = torch.randperm(total, generator=gen, device="cuda")[1:]
    table = torch.zeros(len(need), max(need) + 1, dtype=torch.int64, device="cuda")
    row = torch.repeat_interleave(torch.arange(len(need)), torch.tensor(need)).to("cuda")
    first = torch.tensor([0] + need[:-1]).cumsum(0).to("cuda")
    table[row, torch.arange(total - 1, device="cuda") - first[row]] = order
    return table.to(torch.int32), total


def _step_plan(case, s, contexts, news, gen):
    table, pages = _pages(case, contexts, news, gen)
    s |= {"table": table, "lengths": torch.tensor(contexts, dtype=torch.int32, device="cuda"),
          "cu": torch.tensor([0] + news).cumsum(0).to(torch.int32).to("cuda"), "longest": max(news),
          "most": max(c + n for c, n in zip(contexts, news))}
    if own:
        _package()
        from model.mhc_cache import CacheStep
        s["step"] = CacheStep(s["table"], s["lengths"], s["cu"])
    return pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=dev, generator=gen).to(dtype)

    s = {"case": case}
    op = case["op"]
    dt = DTYPES[case.get("dtype", "fp32")]
    if op == "rotate":
        t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        # what q_norm and k_norm leave: unit-scale rows
        if case["fused"]:
            qkv = randn(t, h + 2 * hk, d, dtype=dt)
            q, k = qkv[:, :h], qkv[:, h:h + hk]
        else:
            q, k = randn(t, h, d, dtype=dt), randn(t, hk, d, dtype=dt)
        if case["rows"]:
            q, k = (x.unflatten(0, (case["rows"], t // case["rows"])) for x in (q, k))
            s["positions"] = None
        else:
            s["positions"] = torch.randint(0, case["far"] + 1, (1,), device=dev, generator=gen) + torch.arange(t, device=dev)
        s |= {"q": q.detach().requires_grad_(case["grad"]), "k": k.detach().requires_grad_(case["grad"])}
        if case["grad"]:
            s |= {"dq": randn(*q.shape, dtype=dt), "dk": randn(*k.shape, dtype=dt)}
        _positions_plan(case, s)
        return s
    contexts, news, parents = _steps(case)
    t = sum(news)
    if op in ("append", "attend", "keep"):
        pages = _step_plan(case, s, contexts, news, gen)
        hk, d = case["kv_heads"], case["dim"]
        shape = (pages, case["page"], hk, d)
        if op == "keep":
            shape = (case["layers"], *shape)
        s |= {"keys": randn(*shape, dtype=dt), "values": randn(*shape, dtype=dt)}
    if op == "append":
        s |= {"q": randn(t, case["heads"], d, dtype=dt), "k": randn(t, hk, d, dtype=dt), "v": randn(t, hk, d, dtype=dt)}
        _positions_plan(case, s)
    elif op == "attend":
        s["q"] = randn(t, case["heads"], d, dtype=dt)
        s["mask"] = None
        if case["tree"]:
            s["mask"] = torch.tensor([_signed(x) for p in parents for x in _ancestors(p)[0]], device=dev)
    elif op == "keep":
        rng = random.Random(seed)
        path, kept = [], []
        for p in parents:  # a way down a random tree: every kept token lies behind the one before
            at, way = 0, [0]
            while at < len(p) - 1 and rng.random() < 0.8:
                at = rng.randrange(at + 1, min(at + 9, len(p)))
                way.append(at)
            path += way + [-1] * (len(p) - len(way))
            kept.append(len(way))
        s |= {"path": torch.tensor(path, dtype=torch.int32, device=dev),
              "kept": torch.tensor(kept, dtype=torch.int32, device=dev)}
    elif op == "verify":
        v = case["vocab"]
        # the target's rows, and a draft's that has learnt most of them
        logits = randn(t, v).mul_(2.5)
        target = torch.softmax(logits, -1)
        draft = torch.softmax(logits.add_(randn(t, v).mul_(0.4)), -1)
        del logits
        starts = [sum(news[:b]) for b in range(case["batch"])]
        up = torch.tensor([st + max(p, 0) for st, ps in zip(starts, parents) for p in ps], device=dev)
        if case["draft"]:  # every drafted token drawn from the draft's row of its parent
            tokens = torch.empty(t, dtype=torch.int64, device=dev)
            for a in range(0, t, 64):
                tokens[a:a + 64] = torch.multinomial(draft[up[a:a + 64]], 1, generator=gen)[:, 0]
        else:  # the draft's likeliest tokens, another one for every child of a node
            rank = torch.tensor([sum(ps[i] == ps[j] for i in range(j)) for ps in parents for j in range(len(ps))], device=dev)
            best = torch.stack([r.topk(int(rank.max()) + 1).indices for r in draft])
            tokens = best[up, rank]
            draft = None
        s |= {"target": target, "draft": draft, "tokens": tokens,
              "parents": torch.tensor([p for ps in parents for p in ps], dtype=torch.int32, device=dev),
              "cu": torch.tensor([0] + news).cumsum(0).to(torch.int32).to(dev), "longest": max(news),
              "random": torch.rand(t, device=dev, generator=gen)}
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _turn(x, cos, sin, interleaved, back=False):
    """Rotates the first elements of every head of x (..., heads, D); cos and sin (..., part / 2) with the gain in them.
    `back`: the transposed rotation, which takes a result's gradient to the argument's."""
    n = 2 * cos.shape[-1]
    y = x.detach().float()
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    if back:
        sin = -sin
    a, b = (y[..., 0:n:2], y[..., 1:n:2]) if interleaved else (y[..., :n // 2], y[..., n // 2:n])
    u, w = a * cos - b * sin, b * cos + a * sin
    first = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((first, y[..., n:]), -1).to(x.dtype)


def _angles(s, positions):
    # the product in 64 bits: 32 lose the angle of a far position
    a = positions.double().unsqueeze(-1) * s["inv_freq"]
    return (a.cos() * s["gain"]).float(), (a.sin() * s["gain"]).float()


def _rotate(s):
    case, inter = s["case"], s["case"]["interleaved"]
    positions = s["positions"]
    if positions is None:
        positions = torch.arange(s["q"].shape[1], device="cuda").expand(s["q"].shape[:2])
    cos, sin = _angles(s, positions)
    out = {"q": _turn(s["q"], cos, sin, inter), "k": _turn(s["k"], cos, sin, inter)}
    if case["grad"]:
        out |= {"dq": _turn(s["dq"], cos, sin, inter, True), "dk": _turn(s["dk"], cos, sin, inter, True)}
    return out


def _places(s):
    """Sequence, place within it and page and slot of every new token."""
    t = s["k"].shape[0]
    cu, at = s["cu"].long(), torch.arange(t, device="cuda")
    row = torch.searchsorted(cu[1:].contiguous(), at, right=True)
    place = s["lengths"].long()[row] + at - cu[row]
    size = s["case"]["page"]
    return place, s["table"].long()[row, place // size], place % size


def _append(s):
    inter = s["case"]["interleaved"]
    place, page, slot = _places(s)
    cos, sin = _angles(s, place)
    s["keys"][page, slot] = _turn(s["k"], cos, sin, inter)
    s["values"][page, slot] = s["v"]
    return {"q": _turn(s["q"], cos, sin, inter), "keys": s["keys"], "values": s["values"]}


def _padded(s, x, n, fill=0):
    """(T, ...) -> (B, n, ...) and which places hold a token."""
    cu = s["cu"].long()
    pos = torch.arange(n, device=x.device)
    here = pos[None] < (cu[1:] - cu[:-1])[:, None]
    return x[(cu[:-1, None] + pos[None]).clamp(max=x.shape[0] - 1)], here


def _attend(s):
    """Softmax attention of every sequence's new tokens over its cache, the sequences padded to the longest."""
    case = s["case"]
    h, hk, d, size = case["heads"], case["kv_heads"], case["dim"], case["page"]
    n, most, b = s["longest"], s["most"], case["batch"]
    q, here = _padded(s, s["q"].float(), n)                                  # (B, n, H, D)
    at = torch.arange(most, device="cuda")
    page = s["table"].long()[:, at // size]                                  # (B, L)
    slot = (at % size).expand_as(page)
    k, v = (s[x][page, slot].float().permute(0, 2, 3, 1) for x in ("keys", "values"))  # (B, Hk, D, L)
    length = s["lengths"].long()
    new = at[None] - length[:, None]                                         # which new token a key is, if one
    if s["mask"] is None:
        seen = new[:, None] <= torch.arange(n, device="cuda")[None, :, None]
    else:
        bits, _ = _padded(s, s["mask"], n)
        seen = ((bits[:, :, None] >> new.clamp(0, 63)[:, None]) & 1).bool() & (new < 64)[:, None] | (new < 0)[:, None]
    news = (s["cu"][1:] - s["cu"][:-1]).long()
    seen = (seen & (new < news[:, None])[:, None]).unsqueeze(1)              # (B, 1, n, L)
    q = q.view(b, n, hk, h // hk, d)
    out = torch.empty_like(q)
    for g in range(h // hk):
        x = (q[:, :, :, g].permute(0, 2, 1, 3) @ k).mul_(d ** -0.5).masked_fill_(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        x = x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
        total = x.sum(-1, keepdim=True)
        x = x.div_(torch.where(total > 0, total, torch.ones_like(total)))
        out[:, :, :, g] = (x @ v.transpose(-1, -2)).permute(0, 2, 1, 3)
    return {"out": out.view(b, n, h, d)[here].to(s["q"].dtype)}


def _verify(s):
    """Goes through every sequence's drafted tokens in their order, all sequences at once.  A child of the last kept
    node is kept if random * mass * draft < rest, where rest is what is left of the target's row: what a refused child's
    row of the draft (or, without one, the child itself) covers is taken off.  The next token is drawn from the rest."""
    target, draft, tokens, n = s["target"], s["draft"], s["tokens"], s["longest"]
    t, v = target.shape
    cu = s["cu"].long()
    b = cu.numel() - 1
    rows = torch.arange(b, device="cuda")
    count = cu[1:] - cu[:-1]
    cur, kept = torch.zeros_like(count), torch.ones_like(count)
    path = torch.full((t,), -1, dtype=torch.int32, device="cuda")
    path[cu[:-1]] = 0
    gone, mass = torch.zeros(b, dtype=torch.float64, device="cuda"), torch.ones(b, dtype=torch.float64, device="cuda")
    out = torch.zeros(b, v, dtype=torch.bool, device="cuda")  # tokens that were refused, where there is no draft
    zero = torch.zeros((), dtype=torch.float64, device="cuda")

    def rest():
        p = target[cu[:-1] + cur].double()
        if draft is None:
            return p.masked_fill(out, 0.0)
        return (p - gone[:, None] * draft[cu[:-1] + cur].double()).clamp(min=0.0)

    for j in range(1, n):
        at = cu[:-1] + count.clamp(max=j + 1) - 1
        asked = (j < count) & (s["parents"][at].long() == cur)
        x = tokens[at]
        p = target[cu[:-1] + cur, x].double()
        q = draft[cu[:-1] + cur, x].double() if draft is not None else torch.ones_like(p)
        r = (p - gone * q).clamp(min=0.0) if draft is not None else torch.where(out[rows, x], zero, p)
        take = asked & (s["random"][at].double() * mass * q < r)
        refuse = asked & ~take
        if draft is None:
            out[rows, x] |= refuse
            out &= ~take[:, None]
            mass = torch.where(take, torch.ones_like(mass), torch.where(refuse, mass - r, mass))
        else:
            gone = torch.where(take, torch.zeros_like(gone), torch.where(refuse, gone + mass, gone))
            mass = torch.where(take, torch.ones_like(mass), torch.where(refuse, rest().sum(-1), mass))
        cur = torch.where(take, torch.full_like(cur, j), cur)
        place = torch.where(take, cu[:-1] + kept, at)
        path[place] = torch.where(take, cur.int(), path[place])
        kept = kept + take
    r = rest()
    total = r.sum(-1, keepdim=True)
    whole = target[cu[:-1] + cur].double()
    r = torch.where(total > 0, r, whole)
    total = torch.where(total > 0, total, whole.sum(-1, keepdim=True))
    goal = s["random"][cu[:-1]].double()[:, None] * total
    index = (r.cumsum(-1) <= goal).sum(-1)
    last = torch.where(r > 0, torch.arange(v, device="cuda"), -1).amax(-1)
    return {"path": path, "kept": kept.int(), "next": torch.minimum(index, last)}


def _keep(s):
    """The i-th kept token's rows of every layer go to the i-th place behind the context."""
    size, t = s["case"]["page"], s["path"].shape[0]
    cu, at = s["cu"].long(), torch.arange(t, device="cuda")
    row = torch.searchsorted(cu[1:].contiguous(), at, right=True)
    i = at - cu[row]
    moved = i < s["kept"][row]
    base, table = s["lengths"].long()[row], s["table"].long()
    src = base + torch.where(moved, s["path"].long(), i)
    dst = base + i
    for x in (s["keys"], s["values"]):
        x[:, table[row, dst // size], dst % size] = x[:, table[row, src // size], src % size]
    return {"keys": s["keys"], "values": s["values"]}


# ---------------------------------------------------------------------------
# The repository's entry points
# ---------------------------------------------------------------------------

def _own(s):
    _package()
    case = s["case"]
    if case["op"] == "rotate":
        from model.mhc_rotary import rotate
        q, k = rotate(s["rotary"], s["q"], s["k"], s["positions"])
        if not case["grad"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if case["op"] == "append":
        from model.mhc_cache import append_kv
        q = append_kv(s["keys"], s["values"], s["step"], s["k"], s["v"], q=s["q"], rotary=s["rotary"])
        return {"q": q, "keys": s["keys"], "values": s["values"]}
    if case["op"] == "attend":
        from model.mhc_cache import cached_attention
        return {"out": cached_attention(s["q"], s["keys"], s["values"], s["step"], mask=s["mask"])}
    if case["op"] == "verify":
        from model.mhc_verify import verify_drafts
        path, kept, following = verify_drafts(s["tokens"], s["parents"], s["cu"], s["target"], s["draft"], s["random"])
        return {"path": path, "kept": kept, "next": following}
    from model.mhc_cache import keep_drafts
    keep_drafts(s["keys"], s["values"], s["step"], s["path"], s["kept"])
    return {"keys": s["keys"], "values": s["values"]}


def run(state):
    if own:
        return _own(state)
    return {"rotate": _rotate, "append": _append, "attend": _attend, "verify": _verify,
            "keep": _keep}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    size = 4 if case.get("dtype", "fp32") == "fp32" else 2
    op = case["op"]
    if op == "rotate":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"] * (2 if case["grad"] else 1)
        # every element read and written; an element of the rotated part costs two products and a sum
        return {"bytes": 2 * size * values, "flops": 3 * values}
    contexts, news, _ = _steps(case)
    t, b = sum(news), case["batch"]
    if op == "append":
        values = t * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * size * (values + t * case["kv_heads"] * case["dim"]) + 8 * b, "flops": 3 * values}
    if op == "attend":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        keys = sum(c + n for c, n in zip(contexts, news))
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(contexts, news))
        return {"bytes": 2 * size * (keys * hk * d + t * h * d) + 8 * t + 4 * keys // case["page"], "flops": 4 * d * h * pairs}
    if op == "verify":
        # the row that the next token is drawn from, of the target and (after a refusal) of the draft, and two
        # probabilities of every drafted token
        rows = 2 if case["draft"] else 1
        return {"bytes": 4 * b * case["vocab"] * rows + 28 * t, "flops": 3 * b * case["vocab"] * rows}
    # a kept token's rows read and written; about half of the sequences' new tokens at most
    moved = sum(min(n, 4) for n in news)
    return {"bytes": 4 * size * case["layers"] * moved * case["kv_heads"] * case["dim"] + 8 * t, "flops": 0}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_turn(s, x, positions, sign=1.0):
    """Every pair as a complex number times gain * exp(i * position * frequency)."""
    case = s["case"]
    n = case["part"]
    w, gain = _inv_freq(n, 1e6, case["factor"])
    y = x.detach().double().clone()
    turn = torch.polar(torch.full_like(w, gain).to("cuda").expand(*positions.shape, -1).contiguous(),
                       sign * positions.double()[..., None] * w.to("cuda"))[..., None, :]
    if case["interleaved"]:
        y[..., :n] = torch.view_as_real(torch.view_as_complex(y[..., :n].unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    else:
        z = torch.complex(y[..., :n // 2], y[..., n // 2:n]) * turn
        y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
    return y


def _exact_rotate(s):
    positions = s["positions"]
    if positions is None:
        positions = torch.arange(s["q"].shape[1], device="cuda").repeat(s["q"].shape[0], 1)
    out = {x: _exact_turn(s, s[x], positions) for x in ("q", "k")}
    if s["case"]["grad"]:
        out |= {x: _exact_turn(s, s[x], positions, -1.0) for x in ("dq", "dk")}
    return out


def _walk(s):
    """(sequence, first new token, new tokens, context, the places' pages and slots) of every sequence."""
    size = s["case"]["page"]
    cu, lengths, table = s["cu"].tolist(), s["lengths"].tolist(), s["table"].long()
    for i, (lo, hi, c) in enumerate(zip(cu[:-1], cu[1:], lengths)):
        at = torch.arange(c + hi - lo, device="cuda")
        yield lo, hi, c, table[i][at // size], at % size


def _exact_append(s):
    keys, values = s["keys"].double(), s["values"].double()
    q = torch.empty_like(s["q"], dtype=torch.float64)
    for lo, hi, c, page, slot in _walk(s):
        where = torch.arange(c, c + hi - lo, device="cuda")
        q[lo:hi] = _exact_turn(s, s["q"][lo:hi], where)
        keys[page[c:], slot[c:]] = _exact_turn(s, s["k"][lo:hi], where)
        values[page[c:], slot[c:]] = s["v"][lo:hi].double()
    return {"q": q, "keys": keys, "values": values}


def _exact_attend(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    parents = _steps(case)[2]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    for (lo, hi, c, page, slot), up in zip(_walk(s), parents):
        n = hi - lo
        seen = torch.ones(n, c + n, dtype=torch.bool)
        for i in range(n):
            seen[i, c:] = False
            if case["tree"]:
                j = i
                while j >= 0:
                    seen[i, c + j] = True
                    j = up[j]
            else:
                seen[i, c:c + i + 1] = True
        seen = seen.to("cuda")
        for j in range(case["kv_heads"]):
            k, v = (s[x][page, slot, j].double() for x in ("keys", "values"))
            for h in range(j * group, (j + 1) * group):
                logits = s["q"][lo:hi, h].double() @ k.T / math.sqrt(case["dim"])
                out[lo:hi, h] = torch.softmax(logits.masked_fill(~seen, -math.inf), -1) @ v
    return {"out": out}


def _exact_verify(s):
    """One sequence after another, as one would do it by hand."""
    cu = s["cu"].tolist()
    path, kept, following = [], [], []
    for lo, hi in zip(cu[:-1], cu[1:]):
        tokens, up, u = (s[x][lo:hi].tolist() for x in ("tokens", "parents", "random"))
        node, way = 0, [0]
        rest, mass, base = s["target"][lo].double(), 1.0, s["target"][lo].double()
        off = s["draft"][lo].double() if s["draft"] is not None else None
        for j in range(1, hi - lo):
            if up[j] != node:
                continue
            x = tokens[j]
            chance = float(off[x]) if off is not None else 1.0
            if u[j] * mass * chance < float(rest[x]):
                node = j
                way.append(j)
                rest, mass = s["target"][lo + j].double(), 1.0
                base = rest
                off = s["draft"][lo + j].double() if s["draft"] is not None else None
            elif off is not None:
                rest = (rest - mass * off).clamp(min=0)
                mass = float(rest.sum())
            else:
                rest = rest.clone()
                mass -= float(rest[x])
                rest[x] = 0
        if not float(rest.sum()) > 0:
            rest = base
        total = torch.cumsum(rest, 0)
        beyond = torch.nonzero(total > u[0] * float(total[-1]))
        following.append(int(beyond[0]) if len(beyond) else int(torch.nonzero(rest > 0)[-1]))
        path += way + [-1] * (hi - lo - len(way))
        kept.append(len(way))
    return {"path": torch.tensor(path, dtype=torch.int32), "kept": torch.tensor(kept, dtype=torch.int32),
            "next": torch.tensor(following)}


def _exact_keep(s):
    out = {x: s[x].double() for x in ("keys", "values")}
    for (lo, hi, c, page, slot), n in zip(_walk(s), s["kept"].tolist()):
        way = s["path"][lo:lo + n].long() + c
        for x in out:
            out[x][:, page[c:c + n], slot[c:c + n]] = s[x][:, page[way], slot[way]].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend, "verify": _exact_verify,
            "keep": _exact_keep}[case["op"]](s)
