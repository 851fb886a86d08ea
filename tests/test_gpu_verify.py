"""Verification of drafted tokens against a walk by hand in 64 bits.  The outputs are whole numbers and have to be equal:
the kernel's sums are fp64, so a border between two tokens moves by 1e-15 of the row, and none of the draws here comes so
near to one (the walk by hand asserts it)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from model.mhc_verify import verify_drafts


def by_hand(tokens, parents, cu, target, draft, random, limit=1024):
    v = target.shape[1]
    clean = lambda row: torch.nan_to_num(row.double(), nan=0.0, posinf=torch.inf, neginf=0.0).clamp(min=0)  # noqa: E731
    path = torch.full((len(tokens),), -1, dtype=torch.int32)
    kept, following = [], []
    for lo, hi in zip(cu[:-1], cu[1:]):
        if hi <= lo:
            kept.append(0)
            following.append(-1)
            continue
        node, way, u = 0, [0], random[lo:hi].double().tolist()
        base = rest = clean(target[lo])
        off, mass = (clean(draft[lo]) if draft is not None else None), 1.0
        for j in range(1, min(hi - lo, limit)):
            x, p = int(tokens[lo + j]), int(parents[lo + j])
            if p != node or p >= j or not 0 <= x < v:
                continue
            chance, left = (float(off[x]) if off is not None else 1.0), float(rest[x])
            assert u[j] * mass * chance == left or abs(u[j] * mass * chance - left) > 1e-13 * left
            if u[j] * mass * chance < left:
                node = j
                way.append(j)
                base = rest = clean(target[lo + j])
                off, mass = (clean(draft[lo + j]) if draft is not None else None), 1.0
            elif off is not None:
                rest = (rest - mass * off).clamp(min=0)
                mass = float(rest.sum())
            else:
                mass = max(mass - left, 0.0)
                rest = rest.clone()
                rest[x] = 0
        if not (0 < float(rest.sum()) < torch.inf):
            rest = base
        total = rest.cumsum(0)
        if 0 < float(total[-1]) < torch.inf:
            goal = u[0] * float(total[-1])
            beyond = torch.nonzero((total > goal) & (rest > 0))
            near = (total[rest > 0] - goal).abs().min()
            assert goal == 0 or float(near) > 1e-13 * float(total[-1])
            following.append(int(beyond[0]) if len(beyond) else int(torch.nonzero(rest > 0)[-1]))
        else:
            following.append(-1)
        path[lo:lo + len(way)] = torch.tensor(way, dtype=torch.int32)
        kept.append(len(way))
    return path, torch.tensor(kept, dtype=torch.int32), torch.tensor(following)


def check(tokens, parents, cu, target, draft, random):
    got = verify_drafts(tokens, parents, cu, target, draft, random)
    want = by_hand(tokens.cpu(), parents.cpu(), cu.tolist(), target.cpu(), None if draft is None else draft.cpu(), random.cpu())
    for name, a, b in zip(("path", "kept", "next"), got, want):
        assert torch.equal(a.cpu(), b), name
        assert a.dtype == b.dtype
    return got


def trees(sizes, wide, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        out += [-1] + [int(torch.randint(max(0, j - wide), j, (1,), generator=g)) for j in range(1, n)] if n else []
    return torch.tensor(out, dtype=torch.int32)


def make(sizes, v, wide=3, drawn=True, seed=0, dtype=torch.float32, noise=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = sum(sizes)
    logits = 2 * torch.randn(t, v, device="cuda", generator=g)
    target, draft = logits.softmax(-1), (logits + noise * torch.randn(t, v, device="cuda", generator=g)).softmax(-1)
    parents = trees(sizes, wide, seed)
    cu = torch.tensor([0] + sizes).cumsum(0).to(torch.int32)
    start = torch.repeat_interleave(cu[:-1].long(), torch.tensor(sizes))
    up = (start + parents.clamp(min=0)).cuda()
    source = draft if drawn else target
    tokens = torch.multinomial(source[up], 1, generator=g)[:, 0]
    return (tokens, parents.cuda(), cu.cuda(), target.to(dtype), draft.to(dtype) if drawn else None,
            torch.rand(t, device="cuda", generator=g))


@pytest.mark.parametrize("drawn", (True, False))
@pytest.mark.parametrize("wide", (1, 4, 40))
@pytest.mark.parametrize("v", (1, 7, 500, 6400, 50001))
def test_trees(v, wide, drawn):
    sizes = [1, 2, 17, 33, 64, 5, 40]
    for seed in range(3):
        check(*make(sizes, v, wide, drawn, seed))


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_types(dtype):
    """The probabilities as the type holds them; their rows need not sum to one exactly."""
    for drawn in (True, False):
        check(*make([9, 1, 30], 3001, 3, drawn, 5, dtype))


def test_many_and_few():
    check(*make([3] * 300, 101, 2, seed=1))
    check(*make([4], 150000, 1, seed=2))
    check(*make([1300, 1, 2], 60, 50, False, seed=3, noise=0.1))     # nothing behind a sequence's 1024th row is kept
    # a chain that is kept whole, past the 1024th row
    n, v = 1100, 5
    target = torch.zeros(n, v, device="cuda")
    target[:, 2] = 1
    got = check(torch.full((n,), 2, device="cuda"), torch.arange(-1, n - 1, device="cuda", dtype=torch.int32),
                torch.tensor([0, n], device="cuda", dtype=torch.int32), target, None, torch.full((n,), 0.5, device="cuda"))
    assert got.kept.tolist() == [1024] and got.next.tolist() == [2]


def test_refusals_one_after_another():
    """A node with many children, none of them likely: every refusal goes over the row again."""
    v, n = 3000, 24
    g = torch.Generator(device="cuda").manual_seed(0)
    target = torch.rand(n, v, device="cuda", generator=g).softmax(-1)
    draft = (3 * torch.randn(n, v, device="cuda", generator=g)).softmax(-1)
    parents = torch.tensor([-1] + [0] * (n - 1), dtype=torch.int32, device="cuda")
    tokens = torch.multinomial(draft[:1].expand(n, v), 1, generator=g)[:, 0]
    random = torch.full((n,), 0.999, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    check(tokens, parents, cu, target, draft, random)
    # the same token drafted again and again
    check(torch.full_like(tokens, 5), parents, cu, target, draft, random)
    check(torch.full_like(tokens, 5), parents, cu, target, None, random)
    check(torch.arange(n, device="cuda"), parents, cu, target, None, random)


def test_children_that_use_the_row_up():
    """Without a draft: a row that sums to a little more than 1, all of it refused: a token that it does not hold is not kept."""
    target = torch.zeros(5, 9, device="cuda")
    target[:, 2], target[:, 4] = 0.6, 0.40000004
    cu, parents = torch.tensor([0, 5], dtype=torch.int32, device="cuda"), torch.tensor([-1, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
    random = torch.tensor([0.3, 1.0, 1.0, 1.0, 1.0], device="cuda")  # (1 refuses all that it can; the draw stays off the borders)
    got = check(torch.tensor([0, 2, 4, 7, 7], device="cuda"), parents, cu, target, None, random)
    assert got.kept.tolist() == [1] or got.path[1] == 2   # the second one may be kept: what is left is less than it


def test_empty_sequences_and_rows_of_none():
    tokens, parents, cu, target, draft, random = make([3, 4, 2], 40)
    cu = torch.tensor([1, 1, 4, 4, 8, 8], dtype=torch.int32, device="cuda")
    parents = torch.tensor([9, -1, 0, 1, -1, 0, 0, 1, 7], dtype=torch.int32, device="cuda")
    got = check(tokens, parents, cu, target, draft, random)
    assert got.kept.tolist()[::2] == [0, 0, 0] and got.next.tolist()[::2] == [-1] * 3
    assert got.path[0] == -1 and got.path[8] == -1
    none = torch.tensor([0], dtype=torch.int32, device="cuda")
    got = verify_drafts(tokens, parents, none, target, draft, random)
    assert got.kept.numel() == 0 and (got.path == -1).all()
    got = verify_drafts(tokens[:0], parents[:0], torch.zeros(3, dtype=torch.int32, device="cuda"), target[:0], None, random[:0])
    assert got.kept.tolist() == [0, 0] and got.next.tolist() == [-1, -1] and got.path.numel() == 0


def test_bad_rows_are_never_kept():
    n, v = 8, 30
    target = torch.full((n, v), 1 / v, device="cuda")
    tokens = torch.tensor([0, 31, -1, 3, 2 ** 40, 4, 5, 6], device="cuda")
    parents = torch.tensor([-1, 0, 0, 3, 0, 6, -5, 100], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = check(tokens, parents, cu, target, None, torch.zeros(n, device="cuda"))
    assert got.kept.tolist() == [1]


def test_special_probabilities():
    cu = torch.tensor([0, 2, 4, 6, 8, 10, 12], dtype=torch.int32, device="cuda")
    v = 50
    target = torch.rand(12, v, device="cuda").softmax(-1)
    draft = torch.rand(12, v, device="cuda").softmax(-1)
    parents = torch.tensor([-1, 0] * 6, dtype=torch.int32, device="cuda")
    tokens = torch.arange(12, device="cuda")
    target[0] = 0                                  # nothing to draw from
    target[2, 7], target[2, 9] = float("nan"), -1.0
    target[4, 3] = float("inf")
    target[6] = draft[6]                           # a refusal leaves nothing: the row itself
    target[8] = 0
    target[8, 41] = 1
    draft[10, 11] = 0                              # a token that could not have been drawn
    random = torch.tensor([.3, .999, .2, .999, .5, .999, .5, 1.0, .0, .999, .5, .999], device="cuda")
    got = check(tokens, parents, cu, target, draft, random)
    assert got.next[0] == -1 and got.next[4] == 41 and got.kept[5] == 2
    assert got.next[2] == -1 or got.kept[2] == 2   # an infinite sum, unless the child was kept


def test_ends_of_the_range():
    """0 takes the first token with anything, 1 - 2^-24 the last but for a part in 2^24, 1 the last one."""
    v = 20000
    target = torch.zeros(3, v, device="cuda")
    target[:, 77], target[:, 19000] = 0.5, 0.5
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    random = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0], device="cuda")
    got = verify_drafts(torch.zeros(3, dtype=torch.int64, device="cuda"), torch.full((3,), -1, dtype=torch.int32, device="cuda"), cu, target,
                        None, random)
    assert got.next.tolist() == [77, 19000, 19000]


def test_strides():
    tokens, parents, cu, target, draft, random = make([5, 9], 333, seed=9)
    wide = torch.full((14, 400), float("nan"), device="cuda")
    wide[:, :333] = target
    turned = draft.t().contiguous().t()
    check(tokens, parents, cu, wide[:, :333], turned, random)
    check(tokens.repeat_interleave(2)[::2], parents.repeat_interleave(2)[::2], cu, target, draft, random.repeat_interleave(2)[::2])


def test_as_if_the_target_had_drawn():
    """One row, three children drawn one after another: over many sequences the first token behind the row follows the
    target, within five standard deviations of a count."""
    v, b = 12, 40000
    g = torch.Generator(device="cuda").manual_seed(3)
    p = (1.5 * torch.randn(v, device="cuda", generator=g)).softmax(-1)
    q = (1.5 * torch.randn(v, device="cuda", generator=g)).softmax(-1)
    tokens = torch.multinomial(q, 4 * b, replacement=True, generator=g)
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda").repeat(b)
    cu = torch.arange(0, 4 * b + 1, 4, dtype=torch.int32, device="cuda")
    got = verify_drafts(tokens, parents, cu, p.expand(4 * b, v).contiguous(), q.expand(4 * b, v).contiguous(),
                        torch.rand(4 * b, device="cuda", generator=g))
    second = got.path.view(b, 4)[:, 1].long()
    first = torch.where(second >= 0, tokens.view(b, 4).gather(1, second.clamp(min=0)[:, None])[:, 0], got.next)
    count = torch.bincount(first, minlength=v).double()
    sigma = (b * p.double() * (1 - p.double())).sqrt()
    assert ((count - b * p.double()).abs() < 5 * sigma).all()
    assert 0 < (second >= 0).sum() < b


def test_captured_and_repeatable():
    a = list(make([6, 20, 11], 7001, seed=11))
    want = verify_drafts(*a)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(want, verify_drafts(*a)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = verify_drafts(*a)
    a[5].copy_(torch.rand(37, device="cuda"))
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(verify_drafts(*a), got))


def test_refused():
    tokens, parents, cu, target, draft, random = make([3, 4], 40)
    for bad in (dict(tokens=tokens.int()), dict(parents=parents.long()), dict(target=target.double()), dict(draft=draft.half()),
                dict(random=random.double()), dict(cu=cu.long())):
        with pytest.raises(TypeError):
            verify_drafts(*({"tokens": tokens, "parents": parents, "cu": cu, "target": target, "draft": draft, "random": random} | bad).values())
    for bad in (dict(tokens=tokens[1:]), dict(parents=parents[1:]), dict(target=target[:, 0]), dict(draft=draft[:, 1:]), dict(random=random[1:]),
                dict(cu=cu[:0]), dict(cu=cu[None])):
        with pytest.raises(ValueError):
            verify_drafts(*({"tokens": tokens, "parents": parents, "cu": cu, "target": target, "draft": draft, "random": random} | bad).values())
    with pytest.raises(RuntimeError, match="CUDA"):
        verify_drafts(tokens, parents, cu, target, draft, random.cpu())


def test_numbers_outside_their_range():
    """Without a draft: 3 refuses a child that has more than is left of the mass, which would fall below 0 then, and 2 times
    that is less than the 0 of a token that the row does not hold: it must not be kept for it.  (With numbers below 1 a
    refused child never has more than the mass.)"""
    target = torch.zeros(4, 9, device="cuda")
    target[:, 2], target[:, 4] = 0.75, 0.5  # a row that sums to more than 1
    cu, parents = torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    random = torch.tensor([0.3, 1.0, 3.0, 2.0], device="cuda")
    got = check(torch.tensor([0, 2, 4, 7], device="cuda"), parents, cu, target, None, random)
    assert got.path.tolist() == [0, -1, -1, -1] and got.kept.tolist() == [1] and got.next.tolist() == [2]
