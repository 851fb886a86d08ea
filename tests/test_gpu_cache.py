"""The paged cache and the attention over it against definitions in 64 bits: types, head layouts, page sizes, lengths from
nothing to long, trees and pieces of prompts, strides, pages that do not exist, NaN in places that nobody sees.

Tolerances.  u = 2^-24 (fp32), 2^-11 (fp16), 2^-8 (bf16); an error is the 2-norm of the difference over the 2-norm of the
exact result.
 * attention, 16 bits: one rounding of every P before the second product and one of the result: 2 u (as for the packed
   attention); fp32: (D + keys) roundings of mixed signs, under 64 u for the lengths here.
 * where a value is held against its exact one by itself (rows that see one key): one rounding of the result and, for 16
   bits, none of P, which is 2^0 or 2^10 there.
 * what is moved or appended unrotated is the same bits; rotated keys are the same bits as ``rotate``'s.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from model import _native as nat
    from model.mhc_attention import packed_attention
    from model.mhc_cache import CacheStep, PagedCache, append_kv, cached_attention, keep_drafts, tree_mask
    from model.mhc_rotary import Rotary, rotate
    from model.mhc_verify import verify_drafts

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
OUT = {torch.float32: 64, torch.float16: 2, torch.bfloat16: 2}
NAN = float("nan")


def err(got, ref):
    assert got.shape == ref.shape
    assert torch.isfinite(got).all()
    n = ref.norm().item()
    d = (got.double() - ref).norm().item()
    return d / n if n else d


def table_of(lengths, page, seed=0, spare=2, columns=2):
    """Pages in random order, the table `columns` wider than the longest sequence needs; its rest points nowhere.  (Where
    the table has room for more than 512 keys, sequences may be shared out among blocks.)"""
    need = [-(-max(n, 0) // page) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), max(need + [0]) + columns), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table.cuda(), total


def make(lens, news, h, hk, d, page, dtype, seed=0, fill=NAN, columns=2):
    """A cache with what the sequences hold, `fill` everywhere else, and the step."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    table, pages = table_of([a + b for a, b in zip(lens, news)], page, seed, columns=columns)
    keys = torch.full((pages, page, hk, d), fill, device="cuda", dtype=dtype)
    values = torch.full_like(keys, fill)
    k, v = [], []
    for b, n in enumerate(a + c for a, c in zip(lens, news)):
        k.append(torch.randn(n, hk, d, device="cuda", generator=g).to(dtype))
        v.append(torch.randn(n, hk, d, device="cuda", generator=g).to(dtype))
        at = torch.arange(n, device="cuda")
        where = table[b].long()[at // page], at % page
        keys[where], values[where] = k[-1], v[-1]
    t = sum(news)
    q = torch.randn(t, h, d, device="cuda", generator=g).to(dtype)
    step = CacheStep(table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                     torch.tensor([0] + list(news)).cumsum(0).to(torch.int32).cuda())
    return q, keys, values, step, k, v


def reference(q, k, v, lens, news, mask=None, scale=None, hole=None):
    """Sequence by sequence in fp64; hole(b, key): keys that do not exist."""
    t, h, d = q.shape
    out = torch.zeros(t, h, d, dtype=torch.float64, device=q.device)
    lo = 0
    for b, (c, n) in enumerate(zip(lens, news)):
        if n == 0:
            continue
        kk, vv = k[b].double(), v[b].double()
        keys = torch.arange(kk.shape[0], device=q.device)
        new = keys - c
        if mask is None:
            seen = new[None] <= torch.arange(n, device=q.device)[:, None]
        else:
            seen = (new < 0)[None] | (((mask[lo:lo + n, None] >> new.clamp(0, 63)[None]) & 1).bool() & (new < 64)[None])
        if hole is not None:
            seen = seen & ~torch.tensor([hole(b, int(x)) for x in keys], dtype=torch.bool, device=q.device)[None]
        r = h // kk.shape[1]
        s = torch.einsum("ihd,jhd->hij", q[lo:lo + n].double(), kk.repeat_interleave(r, 1)) * (d ** -0.5 if scale is None else scale)
        p = s.masked_fill(~seen[None], -math.inf).softmax(-1).nan_to_num(0.0)
        vv = torch.where(seen.any(0)[:, None, None], vv, torch.zeros_like(vv))
        out[lo:lo + n] = torch.einsum("hij,jhd->ihd", p, vv.repeat_interleave(r, 1))
        lo += n
    return out


def random_trees(news, seed=0, wide=4):
    g = torch.Generator().manual_seed(seed)
    parents = [p for n in news for p in ([-1] + [int(torch.randint(max(0, j - wide), j, (1,), generator=g)) for j in range(1, n)] if n else [])]
    cu = torch.tensor([0] + list(news)).cumsum(0).to(torch.int32).cuda()
    mask, depth = tree_mask(torch.tensor(parents, dtype=torch.int32, device="cuda"), cu)
    return mask, depth, torch.tensor(parents, dtype=torch.int32, device="cuda"), cu


def check(lens, news, h, hk, d, page, dtype, mask=None, seed=0, scale=None):
    q, keys, values, step, k, v = make(lens, news, h, hk, d, page, dtype, seed)
    got = cached_attention(q, keys, values, step, mask=mask, scale=scale)
    assert got.dtype == dtype and got.is_contiguous()
    e = err(got, reference(q, k, v, lens, news, mask, scale))
    assert e < OUT[dtype] * U[dtype], e / U[dtype]
    return got


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 130, 700, 5]


@pytest.mark.parametrize("h,hk,d", ((8, 4, 96), (8, 8, 64), (5, 5, 32), (6, 2, 128), (8, 1, 80), (3, 1, 40), (16, 1, 64), (12, 6, 8)))
@pytest.mark.parametrize("dtype", tuple(U))
def test_single_tokens(dtype, h, hk, d):
    for page in (16, 64, 7):
        check(LENS, [1] * len(LENS), h, hk, d, page, dtype, seed=d)


@pytest.mark.parametrize("page", (8, 16, 17, 48, 64, 128, 256))
@pytest.mark.parametrize("dtype,h,hk,d", ((torch.bfloat16, 8, 4, 96), (torch.float16, 8, 2, 128), (torch.bfloat16, 4, 4, 64), (torch.float32, 4, 2, 64),
                                          (torch.float16, 9, 3, 32)))
def test_trees(dtype, h, hk, d, page):
    news = [1, 64, 0, 33, 2, 17, 40, 64]
    lens = [100, 0, 5, 63, 200, 1, 129, 640]
    mask = random_trees(news)[0]
    check(lens, news, h, hk, d, page, dtype, mask)
    check(lens, news, h, hk, d, page, dtype)


@pytest.mark.parametrize("dtype,h,hk,d,page", ((torch.bfloat16, 8, 4, 96, 32), (torch.float16, 2, 2, 128, 17), (torch.float32, 3, 1, 40, 64),
                                               (torch.bfloat16, 4, 1, 72, 128), (torch.bfloat16, 7, 7, 20, 16)))
def test_pieces_of_prompts(dtype, h, hk, d, page):
    """More new tokens than a mask has bits, over empty and filled caches."""
    check([0, 300, 77, 1], [200, 65, 3, 129], h, hk, d, page, dtype)


@pytest.mark.parametrize("rows", (1, 3, 8, 9, 16, 17, 32, 33, 64, 128, 129, 300))
@pytest.mark.parametrize("page", (16, 24))
def test_rows_of_an_item(rows, page):
    """One key head, one query head: as many rows as new tokens, through every kernel."""
    for dtype in (torch.bfloat16, torch.float32):
        check([90, 0, 511], [rows] * 3, 1, 1, 64, page, dtype)


def test_odd_heads_without_wide_copies():
    for d in (1, 3, 9, 33, 60, 127):
        check([0, 40, 130], [2, 1, 9], 4, 2, d, 16, torch.bfloat16)
        check([0, 40, 130], [2, 1, 9], 4, 2, d, 16, torch.float32)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
def test_cuda_cores_for_every_type(dtype):
    before = nat.lib().mhc_set_path_policy(nat.PATH_GENERIC)
    try:
        check([0, 40, 130, 900], [2, 1, 30, 1], 8, 2, 96, 16, dtype)
        check([0, 40, 130, 900], [1, 1, 1, 1], 8, 4, 64, 16, dtype)
    finally:
        nat.lib().mhc_set_path_policy(before)


@pytest.mark.parametrize("dtype,new,page", ((torch.bfloat16, 1, 64), (torch.float16, 1, 64), (torch.bfloat16, 16, 16), (torch.bfloat16, 40, 17),
                                            (torch.float32, 1, 64)))
def test_long(dtype, new, page):
    """One long sequence beside short ones: its keys are shared out among the blocks."""
    check([60000, 3, 9000], [new, 1, new], 4, 2, 64, page, dtype)


def test_many_sequences():
    """More than are looked up in shared memory; most of them without a new token."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 200, (300,), generator=g).tolist()
    for news in ([1] * 300, [3 if b % 7 == 0 else 0 for b in range(300)], [20 if b % 50 == 49 else 0 for b in range(300)]):
        check(lens, news, 4, 2, 64, 16, torch.bfloat16)


def test_nothing_to_see():
    """Masks that leave a row empty, caches without a token, rows of no sequence, no rows at all: 0 (or nothing)."""
    for dtype, page in ((torch.bfloat16, 16), (torch.bfloat16, 17), (torch.float32, 16)):
        for new, columns in ((1, 2), (5, 2), (40, 2), (1, 70), (5, 70), (40, 70)):
            lens, news = [0, 30], [new, new]
            q, keys, values, step, k, v = make(lens, news, 4, 2, 64, page, dtype, columns=columns)
            mask = torch.zeros(2 * new, dtype=torch.int64, device="cuda")
            mask[new + new // 2:] = -1
            got = cached_attention(q, keys, values, step, mask=mask)
            ref = reference(q, k, v, lens, news, mask)
            assert (got[:new] == 0).all() and (ref[:new] == 0).all()
            assert err(got, ref) < OUT[dtype] * U[dtype]
    q, keys, values, step, k, v = make([50, 20], [4, 3], 4, 2, 64, 16, torch.bfloat16)
    # two rows before the first sequence, three behind the last
    wide = torch.randn(12, 4, 64, device="cuda").bfloat16()
    wide[2:9] = q
    got = cached_attention(wide, keys, values, CacheStep(step.page_table, step.lengths, step.cu_tokens + 2))
    assert (got[:2] == 0).all() and (got[9:] == 0).all()
    assert torch.equal(got[2:9], cached_attention(q, keys, values, step))
    none = CacheStep(step.page_table[:0], step.lengths[:0], step.cu_tokens[:1])
    assert (cached_attention(q, keys, values, none) == 0).all()
    assert cached_attention(q[:0], keys, values, CacheStep(step.page_table, step.lengths, torch.zeros_like(step.cu_tokens))).shape == (0, 4, 64)
    empty = CacheStep(step.page_table[:, :0], step.lengths, step.cu_tokens)
    assert (cached_attention(q, keys, values, empty) == 0).all()
    assert (cached_attention(q, keys[:0], values[:0], step) == 0).all()


@pytest.mark.parametrize("dtype,page", ((torch.bfloat16, 16), (torch.bfloat16, 17), (torch.float16, 64), (torch.float32, 16)))
@pytest.mark.parametrize("new", (3, 24, 60))
@pytest.mark.parametrize("columns", (2, 90))
def test_pages_that_do_not_exist(dtype, page, new, columns):
    lens, news = [200, 90], [new, new]
    q, keys, values, step, k, v = make(lens, news, 4, 2, 64, page, dtype, columns=columns)
    table = step.page_table.clone()
    table[0, 3], table[0, 0], table[1, 2] = -1, keys.shape[0], 2 ** 31 - 1
    gone = {(0, 3), (0, 0), (1, 2)}
    got = cached_attention(q, keys, values, CacheStep(table, step.lengths, step.cu_tokens))
    ref = reference(q, k, v, lens, news, hole=lambda b, key: (b, key // page) in gone)
    assert err(got, ref) < OUT[dtype] * U[dtype]
    # a table that ends before the sequence does
    short = step.page_table[:, :4].contiguous()
    got = cached_attention(q, keys, values, CacheStep(short, step.lengths, step.cu_tokens))
    ref = reference(q, k, v, lens, news, hole=lambda b, key: key >= 4 * page)
    assert err(got, ref) < OUT[dtype] * U[dtype]


@pytest.mark.parametrize("bad", (NAN, math.inf, -math.inf))
@pytest.mark.parametrize("dtype,page", ((torch.bfloat16, 16), (torch.bfloat16, 17), (torch.float16, 64), (torch.float32, 16)))
@pytest.mark.parametrize("new,group", ((1, 2), (6, 2), (12, 1), (20, 1), (64, 4)))
@pytest.mark.parametrize("columns", (2, 90))
def test_what_is_not_seen_does_not_touch(dtype, page, new, group, bad, columns):
    """A new token whose keys and values hold nothing but `bad`: the rows that see it are lost, the others the same as
    without it.  (The cache's unused places hold NaN in every test here.)"""
    lens, news = [70, 0], [new, new]
    q, keys, values, step, k, v = make(lens, news, 2 * group, 2, 64, page, dtype, columns=columns)
    mask = random_trees(news, wide=3)[0]
    bit = new // 2
    mask[0:new:3] &= ~(1 << bit)
    clean = cached_attention(q, keys, values, step, mask=mask)
    at = lens[0] + bit
    keys[step.page_table[0, at // page], at % page] = bad
    values[step.page_table[0, at // page], at % page] = bad
    got = cached_attention(q, keys, values, step, mask=mask)
    sees = ((mask >> bit) & 1).bool()
    sees[new:] = False
    assert torch.isfinite(got[~sees]).all()
    # (the reference that a row's sums go by may be another one: as near as two results of it can be)
    assert err(got[~sees], clean[~sees].double()) < 2 * OUT[dtype] * U[dtype]
    if math.isnan(bad):
        assert got[sees].isnan().all()


@pytest.mark.parametrize("dtype,page", ((torch.bfloat16, 16), (torch.bfloat16, 17), (torch.float32, 16)))
@pytest.mark.parametrize("new", (2, 12, 40))
@pytest.mark.parametrize("columns", (2, 90))
def test_infinite_values_that_are_seen(dtype, page, new, columns):
    """One element of V: it reaches its column of the rows that see it, with its sign, and nothing else."""
    lens, news = [33], [new]
    q, keys, values, step, k, v = make(lens, news, 2, 1, 64, page, dtype, columns=columns)
    clean = cached_attention(q, keys, values, step)
    at = lens[0] + new // 2
    values[step.page_table[0, at // page], at % page, 0, 5] = -math.inf
    got = cached_attention(q, keys, values, step)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[new // 2:, :, 5] = True
    assert (got[hit] == -math.inf).all()
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("dtype,group,new,lens", ((torch.bfloat16, 2, 8000, 0), (torch.float16, 1, 4000, 37), (torch.bfloat16, 4, 3000, 1000)))
def test_one_infinity_in_a_long_piece(dtype, group, new, lens):
    """One overflowed value among thousands of new tokens: it reaches its column of the rows that see it, and costs what its
    neighbourhood costs, not a search of the whole piece by every row (that took 36 times as long with 2048 tokens, 146 with
    8192, and with longer pieces more than the kernel's other warps wait)."""
    q, keys, values, step, k, v = make([lens], [new], group, 1, 64, 64, dtype, columns=9)

    def timed():
        best = math.inf
        for _ in range(4):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            out = cached_attention(q, keys, values, step)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        return out, best

    clean, usual = timed()
    for bit in (3, new // 2 + 1, new - 1):
        at = lens + bit
        where = step.page_table[0, at // 64], at % 64, 0, 5
        was = values[where].clone()
        values[where] = math.inf
        got, took = timed()
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[bit:, :, 5] = True
        assert (got[hit] == math.inf).all()
        assert torch.equal(got[~hit], clean[~hit])
        assert took < 8 * usual
        values[where] = was
    assert torch.equal(cached_attention(q, keys, values, step), clean)


@pytest.mark.parametrize("dtype,page", ((torch.bfloat16, 16), (torch.float16, 17), (torch.bfloat16, 64), (torch.float32, 16)))
@pytest.mark.parametrize("group,lens", ((1, 0), (3, 70), (8, 5)))
@pytest.mark.parametrize("columns", (1, 90))
def test_lost_tokens_of_a_piece(dtype, page, group, lens, columns):
    """No mask, several tiles of rows: a new token of nothing but NaN is lost with those behind it, one infinity of V reaches
    its column of these rows, and the rows before are as they were, wherever in a tile it lies."""
    new = 300
    q, keys, values, step, k, v = make([lens, 3], [new, 2], 2 * group, 2, 64, page, dtype, columns=columns)
    clean = cached_attention(q, keys, values, step)
    for bit in (0, 1, 63, 64, 127, 128, 130, new - 1):
        at = lens + bit
        where = step.page_table[0, at // page], at % page
        kept = keys[where].clone(), values[where].clone()
        values[where + (1, 7)] = -math.inf
        got = cached_attention(q, keys, values, step)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[bit:new, group:, 7] = True
        assert (got[hit] == -math.inf).all()
        assert torch.equal(got[~hit], clean[~hit])
        keys[where], values[where] = NAN, NAN
        got = cached_attention(q, keys, values, step)
        assert got[bit:new].isnan().all()
        seen = torch.cat((got[:bit], got[new:])), torch.cat((clean[:bit], clean[new:]))
        # (the references that the sums go by may be other ones)
        assert err(seen[0], seen[1].double()) < 2 * OUT[dtype] * U[dtype]
        keys[where], values[where] = kept
    assert torch.equal(cached_attention(q, keys, values, step), clean)


@pytest.mark.parametrize("dtype,page,new", ((torch.bfloat16, 16, 1), (torch.bfloat16, 17, 9), (torch.bfloat16, 16, 30), (torch.float32, 16, 3)))
@pytest.mark.parametrize("columns", (2, 90))
def test_scores_at_the_ends(dtype, page, new, columns):
    lens, news = [40], [new]
    q, keys, values, step, k, v = make(lens, news, 2, 1, 64, page, dtype, columns=columns)
    # one key far above all others, scores up to 1e30: its values come out
    big = torch.zeros_like(q)
    big[..., 0] = 1e15
    at = 7
    k[0][:, :, 0] = -1e15
    k[0][at, :, 0] = 1e15
    n = torch.arange(lens[0] + new, device="cuda")
    keys[step.page_table[0].long()[n // page], n % page] = k[0]
    got = cached_attention(big, keys, values, step)
    assert torch.equal(got, v[0][at].expand_as(got))
    # all of a row's scores -inf: no softmax, NaN, as the formula says; one finite one: its values
    k[0][:, :, 0] = -math.inf
    keys[step.page_table[0].long()[n // page], n % page] = k[0]
    ones = torch.zeros_like(q)
    ones[..., 0] = 1
    assert cached_attention(ones, keys, values, step).isnan().all()
    keys[step.page_table[0, at // page], at % page, :, 0] = -3.0
    assert torch.equal(cached_attention(ones, keys, values, step), v[0][at].expand_as(got))


def test_strides():
    lens, news = [70, 0, 129], [5, 20, 1]
    mask = random_trees(news)[0]
    for new_rows in (1, 0):
        for dtype in (torch.bfloat16, torch.float32):
            n = [1, 1, 1] if new_rows else news
            m = None if new_rows else mask
            q, keys, values, step, k, v = make(lens, n, 4, 2, 64, 16, dtype)
            want = cached_attention(q, keys, values, step, mask=m)
            # keys and values interleaved in one tensor; heads before slots; pages in the innermost order but heads
            both = torch.stack((keys, values), 1)
            assert torch.equal(cached_attention(q, both[:, 0], both[:, 1], step, mask=m), want)
            hnd = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (keys, values)]
            assert torch.equal(cached_attention(q, *hnd, step, mask=m), want)
            turned = [x.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3) for x in (keys, values)]
            ref = reference(q, k, v, lens, n, m)
            assert err(cached_attention(q, *turned, step, mask=m), ref) < OUT[dtype] * U[dtype]
            assert torch.equal(cached_attention(q, keys, hnd[1], step, mask=m), want)
            # rows that begin at odd places
            off = [torch.empty(x.numel() + 3, dtype=dtype, device="cuda")[3:].view_as(x).copy_(x) for x in (keys, values)]
            assert err(cached_attention(q, *off, step, mask=m), ref) < OUT[dtype] * U[dtype]
            # a slice of queries, one row for all heads, a table that is a slice
            fused = torch.cat((q, q), 1)
            assert torch.equal(cached_attention(fused[:, 4:], keys, values, step, mask=m), want)
            one = q[:, :1].expand(-1, 4, -1)
            assert torch.equal(cached_attention(one, keys, values, step, mask=m), cached_attention(one.contiguous(), keys, values, step, mask=m))
            wide = torch.cat((step.page_table, step.page_table), 1)[:, :step.page_table.shape[1]]
            twice = step.page_table.repeat_interleave(2, 1)[:, ::2]
            for t in (wide, twice):
                assert torch.equal(cached_attention(q, keys, values, CacheStep(t, step.lengths, step.cu_tokens), mask=m), want)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements, the sequence on its last pages."""
    pages, page, hk, d = 70000, 128, 4, 128
    keys, values = (torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert keys.numel() > 2 ** 32
    rotary = Rotary(d)
    for new in (1, 30):
        table = (pages - 1 - torch.arange(6, device="cuda", dtype=torch.int32))[None]
        n = 700
        k, v = (torch.randn(n, hk, d, device="cuda").bfloat16() for _ in range(2))
        q = torch.randn(new, 8, d, device="cuda").bfloat16()
        cu = lambda a: torch.tensor([0, a], dtype=torch.int32, device="cuda")  # noqa: E731
        length = lambda a: torch.tensor([a], dtype=torch.int32, device="cuda")  # noqa: E731
        append_kv(keys, values, CacheStep(table, length(0), cu(n - new)), k[:n - new], v[:n - new])
        append_kv(keys, values, CacheStep(table, length(n - new), cu(new)), k[n - new:], v[n - new:])
        got = cached_attention(q, keys, values, CacheStep(table, length(n - new), cu(new)))
        assert err(got, reference(q, [k], [v], [n - new], [new])) < 2 * U[torch.bfloat16]
        path = torch.tensor([0, new - 1][:new] + [-1] * (new - 2), dtype=torch.int32, device="cuda")
        keep_drafts(keys, values, CacheStep(table, length(n - new), cu(new)), path, torch.tensor([min(2, new)], dtype=torch.int32, device="cuda"))
        at = n - new + (1 if new > 1 else 0)
        assert torch.equal(keys[table[0, at // page], at % page], k[n - 1]) and torch.equal(values[table[0, at // page], at % page], v[n - 1])
    del rotary


def test_repeatable_streams_and_graphs():
    for news, mask in (([1] * 20, None), ([40] * 20, random_trees([40] * 20)[0])):
        lens = [b * 97 % 3000 for b in range(20)]
        q, keys, values, step, k, v = make(lens, news, 8, 4, 96, 64, torch.bfloat16)
        want = cached_attention(q, keys, values, step, mask=mask)
        for _ in range(3):
            assert torch.equal(cached_attention(q, keys, values, step, mask=mask), want)
        # two calls at once
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got += [cached_attention(q, keys, values, step, mask=mask) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)
        # two graphs, replayed in turn with other lengths in the step
        lengths = step.lengths.clone()
        live = CacheStep(step.page_table, lengths, step.cu_tokens)
        graphs, outs = [], []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(cached_attention(q, keys, values, live, mask=mask))
            graphs.append(graph)
        for less in (0, 1, 50):
            lengths.copy_((step.lengths - less).clamp(min=0))
            want_now = cached_attention(q, keys, values, live, mask=mask)
            for graph, out in zip(graphs, outs):
                graph.replay()
                assert torch.equal(out, want_now)


@pytest.mark.parametrize("dtype", tuple(U))
@pytest.mark.parametrize("d,part,page,interleaved", ((96, 96, 64, False), (80, 40, 17, True), (42, 6, 16, False), (128, 0, 48, False)))
def test_append(dtype, d, part, page, interleaved):
    lens, news, h, hk = [0, 5, 63, 1000], [3, 0, 70, 1], 6, 2
    q, keys, values, step, _, _ = make(lens, news, h, hk, d, page, dtype)
    rotary = Rotary(part, interleaved=interleaved, gain=1.3) if part else None
    t = sum(news)
    k, v = (torch.randn(t, hk, d, device="cuda").to(dtype) for _ in range(2))
    place = torch.cat([torch.arange(c, c + n) for c, n in zip(lens, news)]).cuda()
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(news)]).cuda()
    for positions in (None, torch.randint(0, 9999, (t,), device="cuda"), torch.randint(0, 9999, (t,), device="cuda", dtype=torch.int32)):
        if rotary is None and positions is not None:
            continue
        kk, vv = keys.clone(), values.clone()
        out = append_kv(kk, vv, step, k, v, q=q if rotary else None, rotary=rotary, positions=positions)
        want_q, want_k = rotate(rotary, q, k, place if positions is None else positions) if rotary else (None, k)
        where = step.page_table.long()[seq, place // page], place % page
        assert torch.equal(kk[where], want_k) and torch.equal(vv[where], v)
        assert out is None if rotary is None else torch.equal(out, want_q)
        rest = torch.ones(kk.shape[:2], dtype=torch.bool, device="cuda")
        rest[where] = False
        same = lambda a, b: torch.equal(a[rest].view(torch.int16 if dtype != torch.float32 else torch.int32),  # noqa: E731
                                        b[rest].view(torch.int16 if dtype != torch.float32 else torch.int32))
        assert same(kk, keys) and same(vv, values)
    if rotary:  # queries left out; caches at other strides, k and v slices of one tensor
        kk, vv = keys.clone(), values.clone()
        assert append_kv(kk, vv, step, k, v, rotary=rotary) is None
        both = torch.stack((keys, values), 1).transpose(2, 3).contiguous().transpose(2, 3)
        qkv = torch.cat((q, k, v), 1)
        got = append_kv(both[:, 0], both[:, 1], step, qkv[:, h:h + hk], qkv[:, h + hk:], q=qkv[:, :h], rotary=rotary)
        assert torch.equal(both[:, 0].nan_to_num(9), kk.nan_to_num(9)) and torch.equal(both[:, 1].nan_to_num(9), vv.nan_to_num(9))
        assert torch.equal(got, rotate(rotary, q, k, place)[0])


def test_append_where_there_is_no_place():
    """Rows of no sequence, places behind the table, negative lengths and pages that are none: nothing is written."""
    rotary = Rotary(32)
    keys, values = torch.zeros(4, 8, 2, 32, device="cuda"), torch.zeros(4, 8, 2, 32, device="cuda")
    table = torch.tensor([[0, -1], [4, 2], [3, 1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([6, 6, -2], dtype=torch.int32, device="cuda")
    cu = torch.tensor([1, 5, 16, 20], dtype=torch.int32, device="cuda")
    k, v, q = (torch.randn(22, n, 32, device="cuda") for n in (2, 2, 4))
    out = append_kv(keys, values, CacheStep(table, lengths, cu), k, v, q=q, rotary=rotary)
    want = torch.zeros_like(values)
    want[0, 6], want[0, 7] = v[1], v[2]            # sequence 0: the rest would go to page -1
    for i in range(8):
        want[2, i] = v[5 + 2 + i]                  # sequence 1: two to page 4, eight to page 2, one behind the table
    want[3, 0], want[3, 1] = v[18], v[19]          # sequence 2 begins at place -2
    assert torch.equal(values, want)
    assert (keys.abs().sum((-1, -2)) > 0).eq(want.abs().sum((-1, -2)) > 0).all()
    assert (out[0] == 0).all() and (out[20:] == 0).all() and (out[1:20].abs().sum((-1, -2)) > 0).all()


@pytest.mark.parametrize("dtype,d,page", ((torch.bfloat16, 96, 64), (torch.float32, 33, 17), (torch.float16, 40, 8)))
@pytest.mark.parametrize("layers", (0, 1, 5))
def test_keep(dtype, d, page, layers):
    lens, news = [0, 7, 100, 63, 5], [40, 1, 12, 30, 0]
    table, pages = table_of([a + b for a, b in zip(lens, news)], page)
    shape = (layers, pages, page, 2, d) if layers else (pages, page, 2, d)
    keys, values = torch.randn(shape, device="cuda").to(dtype), torch.randn(shape, device="cuda").to(dtype)
    ways = [[0, 1, 2, 5, 6, 7, 8, 9, 10, 20, 21, 22, 23, 24, 39], [0], [0, 11], list(range(30)), []]
    path = torch.tensor([x for w, n in zip(ways, news) for x in w + [-1] * (n - len(w))], dtype=torch.int32, device="cuda")
    step = CacheStep(table, torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda())
    want = keys.clone(), values.clone()
    for x, src in zip(want, (keys, values)):
        for b, w in enumerate(ways):
            for i, p in enumerate(w):
                at, to = lens[b] + p, lens[b] + i
                x[..., table[b, to // page], to % page, :, :] = src[..., table[b, at // page], at % page, :, :]
    keep_drafts(keys, values, step, path, torch.tensor([len(w) for w in ways], dtype=torch.int32, device="cuda"))
    assert torch.equal(keys, want[0]) and torch.equal(values, want[1])
    # a path that is none: more kept than there are, rows past the tree, backwards
    path.copy_(torch.randint(-3, 60, path.shape))
    before = keys.clone()
    keep_drafts(keys, values, step, path, torch.full((5,), 10 ** 6, dtype=torch.int32, device="cuda"))
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(news):
        at = torch.arange(lens[b], lens[b] + n, device="cuda")
        used[table[b].long()[at // page], at % page] = True
    if layers:
        assert torch.equal(keys[:, ~used], before[:, ~used])
    else:
        assert torch.equal(keys[~used], before[~used])


def test_tree_mask():
    news = [64, 1, 0, 7, 33]
    mask, depth, parents, cu = random_trees(news, seed=3, wide=64)
    at = 0
    for n in news:
        bits, deep = [], []
        for j in range(n):
            p = int(parents[at + j])
            bits.append((1 << j) | (bits[p] if p >= 0 else 0))
            deep.append(deep[p] + 1 if p >= 0 else 0)
        assert [int(x) & (2 ** 64 - 1) for x in mask[at:at + n]] == bits and depth[at:at + n].tolist() == deep
        at += n
    chain = torch.arange(-1, 63, dtype=torch.int32, device="cuda")
    mask, depth = tree_mask(chain, torch.tensor([0, 64], dtype=torch.int32, device="cuda"))
    assert depth.tolist() == list(range(64)) and int(mask[63]) == -1


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_the_operators_together(dtype):
    """An answer with drafted trees, step by step through the cache, against attention over the kept tokens from scratch."""
    torch.manual_seed(0)
    h, hk, d, page, vocab, batch = 4, 2, 64, 16, 50, 3
    rotary = Rotary(d, 1e4)
    wq, wk, wv, wo = (torch.randn(vocab if i < 3 else h * d, n, device="cuda") * s for i, (n, s) in
                      enumerate(((h * d, 1.0), (hk * d, 1.0), (hk * d, 1.0), (vocab, 0.2))))
    wq, wk, wv = (x.to(dtype) for x in (wq, wk, wv))
    cache = PagedCache(1, 60, page, hk, d, dtype)
    table = torch.randperm(60, device="cuda").to(torch.int32).view(batch, 20)
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    text = [torch.randint(vocab, (n,), device="cuda") for n in (5, 40, 17)]

    def layer(tokens, step, **kw):
        t = tokens.numel()
        q = append_kv(cache.keys[0], cache.values[0], step, wk[tokens].view(t, hk, d), wv[tokens].view(t, hk, d), q=wq[tokens].view(t, h, d),
                      rotary=rotary, positions=kw.get("positions"))
        return cached_attention(q, cache.keys[0], cache.values[0], step, mask=kw.get("mask"))

    def scratch(tokens):
        t = tokens.numel()
        q, k = rotate(rotary, wq[tokens].view(1, t, h, d), wk[tokens].view(1, t, hk, d))
        return packed_attention(q, k, wv[tokens].view(1, t, hk, d))[0]

    cu = torch.tensor([0] + [len(x) for x in text]).cumsum(0).to(torch.int32).cuda()
    out = layer(torch.cat(text), CacheStep(table, lengths, cu))
    last = (out[cu[1:].long() - 1].flatten(1).float() @ wo).argmax(-1)
    lengths = lengths + cu.diff()
    kept_any = 0
    for i in range(6):
        news = [1 + (i * 5 + b * 7) % 12 for b in range(batch)]
        mask, depth, parents, cu = random_trees(news, seed=i, wide=3)
        tokens = torch.randint(vocab, (sum(news),), device="cuda")
        tokens[cu[:-1].long()] = last
        step = CacheStep(table, lengths, cu)
        out = layer(tokens, step, positions=lengths.repeat_interleave(cu.diff()) + depth, mask=mask)
        target = (out.flatten(1).float() @ wo).softmax(-1)
        path, kept, last = verify_drafts(tokens, parents, cu, target, torch.full_like(target, 1 / vocab), torch.rand(sum(news), device="cuda"))
        keep_drafts(cache.keys, cache.values, step, path, kept)
        lengths = lengths + kept
        for b in range(batch):
            lo, n = int(cu[b]), int(kept[b])
            way = lo + path[lo:lo + n].long()
            text[b] = torch.cat((text[b], tokens[way]))
            want = scratch(text[b])[-n:]
            # both are roundings of the same attention; keys are the same bits
            assert err(out[way], want.double()) < 2 * OUT[dtype] * U[dtype]
            kept_any += n - 1
        assert lengths.tolist() == [len(x) for x in text]
    assert kept_any > 0


def test_decoder_over_the_cache():
    """The benchmark's decoder token by token and by trees over the cache against its forward over the whole text.  fp32
    weights: the two differ by roundings of 2^-24 through two layers of sums of a few hundred, under 2^-24 * 2^9."""
    import bench
    torch.manual_seed(1)
    m = bench._build_decoder(moe=False, dev=torch.device("cuda"), hidden=256, layers=2, heads=4, kv_heads=2, inter=512, vocab=512, dtype=torch.float32,
                             native_ops=True).eval()
    ids = torch.randint(512, (2, 50), device="cuda")
    with torch.no_grad():
        want = m(ids)
        cache = PagedCache(2, 10, 16, 2, 64, torch.float32)
        table = torch.arange(10, device="cuda", dtype=torch.int32).view(2, 5)
        lengths, got = torch.zeros(2, dtype=torch.int32, device="cuda"), []
        for lo, hi in ((0, 30), (30, 31), (31, 32), (32, 45), (45, 50)):
            cu = torch.tensor([0, hi - lo, 2 * (hi - lo)], dtype=torch.int32, device="cuda")
            got.append(m(ids[:, lo:hi].flatten(), cache, CacheStep(table, lengths, cu)).view(2, hi - lo, -1))
            lengths = lengths + (hi - lo)
        got = torch.cat(got, 1)
    assert (got - want).norm() / want.norm() < 2.0 ** -15


def test_decode_workload():
    """The command runs and reports."""
    import json
    import os
    import subprocess
    import sys

    from conftest import ROOT
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--workload", "decode", "--steps", "2", "--warmup", "3"], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads(r.stdout.strip().splitlines()[-1])
    assert line["value"] > 0 and 1 <= line["config"]["kept_per_step_and_sequence"] <= 16


def test_offsets_and_lengths_that_are_none():
    """Nothing is said of what comes out, only that every access stays inside: the cache keeps its bits where no place is, and
    later calls are as ever."""
    g = torch.Generator().manual_seed(5)
    for new, columns in ((1, 2), (9, 80), (40, 80)):
        q, keys, values, step, k, v = make([40, 9, 100], [new] * 3, 4, 2, 64, 16, torch.bfloat16, columns=columns)
        want = cached_attention(q, keys, values, step)
        t = q.shape[0]
        kk, vv = (torch.randn(t, 2, 64, device="cuda").bfloat16() for _ in range(2))
        for _ in range(12):
            cu = torch.randint(-2 ** 31, 2 ** 31 - 1, (4,), generator=g)
            cu = (cu if _ % 2 else cu % (2 * t + 1)).to(torch.int32).cuda()
            lengths = torch.randint(-2 ** 31, 2 ** 31 - 1, (3,), generator=g).to(torch.int32).cuda() if _ % 3 else step.lengths
            table = torch.randint(-2 ** 31, 2 ** 31 - 1, step.page_table.shape, generator=g).to(torch.int32).cuda() if _ % 4 else step.page_table
            bad = CacheStep(table, lengths, cu)
            mask = torch.randint(-2 ** 63, 2 ** 63 - 1, (t,), generator=g).cuda()
            cached_attention(q, keys, values, bad, mask=mask if new < 64 and _ % 2 else None)
            spare = keys.clone(), values.clone()
            append_kv(*spare, bad, kk, vv, q=q, rotary=Rotary(64))
            keep_drafts(*spare, bad, torch.randint(-2 ** 31, 2 ** 31 - 1, (t,), generator=g).to(torch.int32).cuda(),
                        torch.randint(-2 ** 31, 2 ** 31 - 1, (3,), generator=g).to(torch.int32).cuda())
        assert torch.equal(cached_attention(q, keys, values, step), want)


def test_refused():
    q, keys, values, step, k, v = make([9, 3], [2, 1], 4, 2, 32, 8, torch.bfloat16)
    kk, vv = torch.zeros(3, 2, 32, device="cuda").bfloat16(), torch.zeros(3, 2, 32, device="cuda").bfloat16()
    path, kept = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    rotary = Rotary(32)
    swap = lambda **x: step._replace(**x)  # noqa: E731
    for bad in (lambda: cached_attention(q.float(), keys, values, step), lambda: cached_attention(q, keys, values.float(), step),
                lambda: cached_attention(q, keys, values, swap(lengths=step.lengths.long())), lambda: cached_attention(q, keys, values, swap(page_table=step.page_table.long())),
                lambda: cached_attention(q, keys, values, step, mask=torch.zeros(3, dtype=torch.int32, device="cuda")),
                lambda: append_kv(keys, values, step, kk.float(), vv), lambda: append_kv(keys, values, step, kk, vv, q=q.float(), rotary=rotary),
                lambda: append_kv(keys, values, step, kk, vv, rotary=rotary, positions=torch.zeros(3, device="cuda")),
                lambda: keep_drafts(keys, values, step, path.long(), kept), lambda: keep_drafts(keys, values, step, path, kept.long()),
                lambda: cached_attention(q.double(), keys.double(), values.double(), step)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: cached_attention(q[:, :3], keys, values, step), lambda: cached_attention(q[..., :16], keys, values, step),
                lambda: cached_attention(q[0], keys, values, step), lambda: cached_attention(q, keys, values[1:], step),
                lambda: cached_attention(q, keys[0], values[0], step), lambda: cached_attention(q, keys, values, swap(lengths=step.lengths[1:])),
                lambda: cached_attention(q, keys, values, swap(cu_tokens=step.cu_tokens[1:])), lambda: cached_attention(q, keys, values, swap(page_table=step.page_table[0])),
                lambda: cached_attention(q, keys, values, step, scale=0.0), lambda: cached_attention(q, keys, values, step, scale=math.inf),
                lambda: cached_attention(q, keys, values, step, mask=torch.zeros(2, dtype=torch.int64, device="cuda")),
                lambda: cached_attention(q.repeat(1, 1, 2), keys.repeat(1, 1, 1, 2)[..., ::2], values, step),
                lambda: cached_attention(torch.zeros(3, 4, 160, device="cuda"), torch.zeros(4, 8, 2, 160, device="cuda"), torch.zeros(4, 8, 2, 160, device="cuda"), step),
                lambda: append_kv(keys, values, step, kk[:, :1], vv[:, :1]), lambda: append_kv(keys, values, step, kk, vv, q=q),
                lambda: append_kv(keys, values, step, kk, vv, q=q[:2], rotary=rotary), lambda: append_kv(keys, values, step, kk, vv, rotary=Rotary(64)),
                lambda: append_kv(keys, values, step, kk, vv, rotary=rotary, positions=path[:2]), lambda: keep_drafts(keys, values, step, path[None], kept),
                lambda: keep_drafts(keys, values, step, path, kept[:1]), lambda: keep_drafts(keys[None, None], values[None, None], step, path, kept)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cached_attention(q.cpu(), keys, values, step), lambda: cached_attention(q, keys, values, swap(lengths=step.lengths.cpu())),
                lambda: append_kv(keys, values, step, kk.cpu(), vv)):
        with pytest.raises(RuntimeError, match="CUDA"):
            bad()
    for bad in (lambda: cached_attention(q.clone().requires_grad_(True), keys, values, step), lambda: append_kv(keys, values, step, kk.clone().requires_grad_(True), vv)):
        with pytest.raises(RuntimeError, match="no gradient"):
            bad()
    with torch.no_grad():
        cached_attention(q.clone().requires_grad_(True), keys, values, step)


def test_sizes_that_32_bits_do_not_hold():
    """(Tensors of one element's memory: nothing is allocated before the refusal.)"""
    one = torch.zeros(1, 1, 8, device="cuda", dtype=torch.bfloat16)
    keys = torch.zeros(4, 16, 1, 8, device="cuda", dtype=torch.bfloat16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    step = CacheStep(i32(0, 1)[None], i32(5), i32(0, 1))
    for t, h in ((1 << 27, 32), (1 << 20, 1 << 12), (1, (1 << 32) + 1)):
        with pytest.raises(ValueError, match="rows"):
            cached_attention(one.expand(t, h, 8), keys, keys, step)
    many = one.expand(1, (1 << 32) + 1, 8)
    for bad in (lambda: rotate(Rotary(8), many, one), lambda: rotate(Rotary(8), one, many), lambda: append_kv(keys, keys, step, one, one, q=many, rotary=Rotary(8)),
                lambda: append_kv(keys.expand(4, 16, (1 << 32) + 1, 8), keys.expand(4, 16, (1 << 32) + 1, 8), step, many, many)):
        with pytest.raises(ValueError):
            bad()


def test_expanded_caches():
    """They can be read (one layer's pages for all, one head for all) and not written to."""
    q, keys, values, step, k, v = make([9, 3], [2, 1], 4, 1, 32, 8, torch.bfloat16)
    heads = keys.expand(-1, -1, 2, -1), values.expand(-1, -1, 2, -1)
    got = cached_attention(q, *heads, step)
    want = cached_attention(q, *(x.repeat(1, 1, 2, 1) for x in (keys, values)), step)
    assert err(got, want.double()) <= U[torch.bfloat16]
    kk = torch.zeros(3, 2, 32, device="cuda").bfloat16()
    path, kept = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    layers = keys.expand(3, -1, -1, -1, -1), values.expand(3, -1, -1, -1, -1)
    before = keys.clone(), values.clone()
    for bad in (lambda: append_kv(*heads, step, kk, kk), lambda: append_kv(heads[0], values.repeat(1, 1, 2, 1), step, kk, kk),
                lambda: keep_drafts(*heads, step, path, kept), lambda: keep_drafts(*layers, step, path, kept),
                lambda: append_kv(keys[:1].expand(6, -1, -1, -1), values[:1].expand(6, -1, -1, -1), step, kk[:, :1], kk[:, :1])):
        with pytest.raises(ValueError, match="expanded"):
            bad()
    assert all(torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(before, (keys, values)))
