"""Packed causal attention against its definition in 64 bits: types, head layouts, lengths from nothing to several
tiles, strides, tokens outside of every sequence, gradients against the formula's and against differences.

Tolerances.  u = 2^-24 (fp32), 2^-11 (fp16), 2^-8 (bf16): the largest relative error of one rounding.  An error is
measured as the 2-norm of the difference over the 2-norm of the exact result.
 * out: one rounding of the result and, with 16-bit inputs, one of every P before the second product: 2 u; fp32 adds
   (D + keys) roundings, under 64 u for the lengths here as their signs are mixed.
 * gradients: P, dS and the result are rounded: under 4 u; fp32 under 256 u (two chained sums).
 * where the exact gradient is zero or nearly so (the dq of a sequence of one token, of equal keys), differences of
   sums of D rounded products remain: FLOOR times the size of dO and sqrt(D) is allowed beside the relative bound.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from model import _native as nat
    from model.mhc_attention import packed_attention

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
OUT = {torch.float32: 64, torch.float16: 2, torch.bfloat16: 2}
GRAD = {torch.float32: 256, torch.float16: 4, torch.bfloat16: 4}


def reference(q, k, v, cu, dout=None, scale=None):
    """Sequence by sequence in fp64; tokens outside get zeros."""
    q, k, v = (x.detach().double() for x in (q, k, v))
    t, h, d = q.shape
    hk = k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for lo, hi in zip(cu[:-1], cu[1:]):
        if hi <= lo:
            continue
        qq, kk, vv = (x[lo:hi].clone().requires_grad_(True) for x in (q, k, v))
        kr, vr = kk.repeat_interleave(h // hk, 1), vv.repeat_interleave(h // hk, 1)
        s = torch.einsum("ihd,jhd->hij", qq, kr) * scale
        n = hi - lo
        s = s.masked_fill(torch.ones(n, n, device=q.device).triu(1).bool(), -math.inf)
        o = torch.einsum("hij,jhd->ihd", s.softmax(-1), vr)
        out[lo:hi] = o.detach()
        if dout is not None:
            dq[lo:hi], dk[lo:hi], dv[lo:hi] = torch.autograd.grad(o, (qq, kk, vv), dout[lo:hi].double())
    return out, dq, dk, dv


def err(got, ref):
    assert got.shape == ref.shape
    assert torch.isfinite(got).all()
    n = ref.norm().item()
    d = (got.double() - ref).norm().item()
    return d / n if n else d


def make(t, h, hk, d, dtype, seed=0, fused=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if fused:
        x = torch.randn(t, h + 2 * hk, d, device="cuda", generator=g).to(dtype)
        q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    else:
        q, k, v = (torch.randn(t, n, d, device="cuda", generator=g).to(dtype) for n in (h, hk, hk))
    return q, k, v, torch.randn(t, h, d, device="cuda", generator=g).to(dtype)


def check(cu, h, hk, d, dtype, total=None, fused=False, seed=0, scale=None):
    t = cu[-1] if total is None else total
    q, k, v, do = make(t, h, hk, d, dtype, seed, fused)
    ref = reference(q, k, v, cu, do, scale)
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), scale)
    grads = torch.autograd.grad(out, (q, k, v), do)
    assert err(out, ref[0]) <= OUT[dtype] * U[dtype]
    for g, r in zip(grads, ref[1:]):
        grad_close(g, r, do, dtype)


DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def grad_close(got, want, do, dtype, times=1):
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    floor = 2.0 ** -20 * do.double().norm().item() * do.shape[-1] ** 0.5
    off = (got.double() - want).norm().item()
    assert off <= times * GRAD[dtype] * U[dtype] * want.norm().item() + floor


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", (1, 2, 31, 64, 65, 127, 128, 129, 255, 257, 300, 513))
def test_one_sequence(dtype, length):
    check([0, length], 2, 1, 64, dtype, seed=length)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (1, 7, 8, 16, 32, 40, 64, 72, 80, 96, 100, 112, 128))
def test_head_sizes(dtype, d):
    check([0, 150, 331], 2, 2, d, dtype, seed=d)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk", ((1, 1), (8, 8), (8, 4), (8, 2), (8, 1), (5, 1), (6, 2), (3, 3), (9, 3)))
def test_grouped_heads(dtype, h, hk):
    check([0, 70, 263], h, hk, 96, dtype, seed=h * 10 + hk)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", (
    [1] * 7, [1] * 300, [0, 5, 0, 0, 130, 0], [128, 128, 128], [3, 200, 1, 1, 64, 129, 17], [127, 1, 127, 1],
    [400, 2, 390], [0, 0, 1], list(range(40))))
def test_packed_lengths(dtype, lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    check(cu, 4, 2, 64, dtype, seed=sum(lengths))


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("d", (64, 36))
@pytest.mark.parametrize("lengths,h,hk", (
    ([512, 512], 8, 8), ([1024], 8, 4), ([300] * 7, 4, 4), ([1, 700, 0, 333, 64], 6, 2), ([1900, 1300, 77, 1], 16, 4)))
def test_more_blocks_than_sms(dtype, d, lengths, h, hk):
    """Ordered blocks, one or two for an SM and many, of both heights; shared-out heads.  Random signs: sums of 64
    products and at most 1900 keys are within sqrt(1964) < 64 roundings."""
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    check(cu, h, hk, d, dtype, seed=cu[-1] + d)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (30, 32, 84, 90, 96, 100, 127, 128))
def test_head_sizes_in_blocks_of_both_heights(dtype, d):
    """Every padded head size of the CUDA-core kernels, tiles that are copied and loaded, with enough tiles for blocks of
    64 rows.  Sums of at most 128 products and 1900 keys: sqrt(2028) < 64 roundings."""
    check([0, 1900, 3200, 3277, 3278], 16, 8, d, dtype, seed=d)


@pytest.mark.parametrize("dtype,d", ((torch.float32, 64), (torch.float32, 96), (torch.float32, 98), (torch.bfloat16, 36),
                                     (torch.bfloat16, 100), (torch.bfloat16, 128), (torch.float16, 96)))
@pytest.mark.parametrize("place", ("q", "k", "v", "do"))
def test_non_finite_values_with_many_blocks(dtype, d, place):
    """A NaN among 3278 tokens of 16 heads, blocks of 64 rows on the CUDA cores: it reaches what sees it only."""
    cu, at, h, hk = [0, 1900, 3200, 3277, 3278], 1990, 16, 8
    x = dict(zip(("q", "k", "v", "do"), make(cu[-1], h, hk, d, dtype, 47)))
    want = reference(x["q"], x["k"], x["v"], cu, x["do"])
    x[place][at, 1, 5] = float("nan")
    reach = poisoned(place, "nan", at, 1, 5, cu, h, hk, cu[-1], d)
    y = [x[n].requires_grad_(True) for n in ("q", "k", "v")]
    out = packed_attention(*y, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    grads = torch.autograd.grad(out, y, x["do"])
    for i, (got, ref, bad) in enumerate(zip((out, *grads), want, reach)):
        assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
        off = (got[~bad].double() - ref[~bad]).norm().item()
        assert off <= (OUT if i == 0 else GRAD)[dtype] * U[dtype] * ref[~bad].norm().item()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 36, 96, 128))
@pytest.mark.parametrize("h,hk", ((4, 2), (1, 1), (16, 1)))
def test_a_token_alone_has_no_gradient_but_its_value(dtype, d, h, hk):
    """Its weight is 1 whatever q and k are: dq and dk are exactly 0, and dv is dO summed over the group's heads (its
    weight in the backward comes from the saved log of the sum: 2^-22 of a score of up to 2^5 beside the rounding)."""
    for cu in (list(range(301)), [0, 0, 1], [3, 4, 5, 5]):
        t = cu[-1]
        q, k, v, do = make(t, h, hk, d, dtype, 43)
        x = [y.requires_grad_(True) for y in (q, k, v)]
        out = packed_attention(*x, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        dq, dk, dv = torch.autograd.grad(out, x, do)
        assert torch.equal(out[cu[0]:], v.repeat_interleave(h // hk, 1)[cu[0]:])
        assert torch.count_nonzero(dq) == 0 and torch.count_nonzero(dk) == 0
        want = do.double().view(t, hk, h // hk, d).sum(2)
        want[:cu[0]] = 0
        assert (dv.double() - want).norm() <= (2 * U[dtype] + 2.0 ** -17) * want.norm()
    # and the first token of a longer sequence has no dq
    q, k, v, do = make(200, h, hk, d, dtype, 44)
    x = [y.requires_grad_(True) for y in (q, k, v)]
    out = packed_attention(*x, torch.tensor([0, 150, 200], dtype=torch.int32, device="cuda"))
    assert torch.count_nonzero(torch.autograd.grad(out, x, do)[0][[0, 150]]) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cu,total", (([5, 90], 140), ([0, 130], 131), ([130, 260], 400), ([3, 3, 4], 9), ([0, 0], 5),
                                      ([200, 200], 300)))
def test_tokens_outside_of_every_sequence(dtype, cu, total):
    """They get zeros and give nothing, whatever they hold."""
    h, hk, d = 4, 2, 64
    q, k, v, do = make(total, h, hk, d, dtype, 3)
    out_rows = torch.ones(total, dtype=torch.bool, device="cuda")
    out_rows[cu[0]:cu[-1]] = False
    ref = reference(q, k, v, cu, do)
    for fill in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
        for x in (q, k, v, do):
            x[out_rows] = fill
        a, b, c = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = packed_attention(a, b, c, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        grads = torch.autograd.grad(out, (a, b, c), do)
        for got, want, u in zip((out, *grads), ref, (OUT[dtype], *[GRAD[dtype]] * 3)):
            assert torch.count_nonzero(got[out_rows]) == 0
            assert torch.isfinite(got).all()
            assert (got.double() - want).norm() <= u * U[dtype] * want.norm() + 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_of_the_future_and_of_other_sequences(dtype):
    """Large finite values in places that a token must not see leave it alone."""
    t, h, hk, d = 300, 2, 2, 64
    q, k, v, _ = make(t, h, hk, d, dtype, 5)
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    one = packed_attention(q, k, v, cu)
    k2, v2 = k.clone(), v.clone()
    big = 3e4
    k2[250:], v2[250:] = big, big       # the future of tokens 100..249
    k2[:100], v2[:100] = -big, big      # another sequence
    two = packed_attention(q, k2, v2, cu)
    assert torch.equal(one[100:250], two[100:250])


def poisoned(place, fill, at, head, col, cu, h, hk, t, d):
    """Which entries of out, dq, dk and dv the definition lets a non-finite entry of an input reach."""
    lo, hi = next((a, b) for a, b in zip(cu[:-1], cu[1:]) if a <= at < b)
    m = [torch.zeros(t, n, d, dtype=torch.bool, device="cuda") for n in (h, h, hk, hk)]
    g = h // hk
    if place == "q":      # a row of P
        m[0][at, head] = m[1][at, head] = True
        m[2][lo:at + 1, head // g] = m[3][lo:at + 1, head // g] = True
    elif place == "k":    # every row of P that sees it, for the heads of the group
        m[0][at:hi, head * g:head * g + g] = m[1][at:hi, head * g:head * g + g] = True
        m[2][lo:hi, head] = m[3][lo:hi, head] = True
    elif place == "v":    # a column of those rows of out; D of those rows, and with it dS; not dv
        m[0][at:hi, head * g:head * g + g, col] = True
        m[1][at:hi, head * g:head * g + g] = True
        m[2][lo:hi, head] = True
    else:                 # dO: a row of dS, a column of dv
        m[1][at, head] = True
        m[2][lo:at + 1, head // g] = True
        m[3][lo:at + 1, head // g, col] = True
    return m


NAN_LENGTHS = (([100, 200, 37, 300], 150, 637), ([513, 3, 1, 700], 2, 1300), ([1000], 400, 1000),
               ([60, 1, 1, 200], 60, 262))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 36, 128))
@pytest.mark.parametrize("place,fill", (("q", "nan"), ("k", "nan"), ("v", "nan"), ("v", "inf"), ("v", "-inf")))
@pytest.mark.parametrize("lengths,at,total", NAN_LENGTHS)
def test_non_finite_values_reach_what_sees_them_only(dtype, d, place, fill, lengths, at, total):
    """A NaN or an infinity in one entry of one head: what the formula takes it to is not finite, and everything else,
    in the same tiles, of later and of earlier tokens of the same sequence, is as without it."""
    h, hk, col = 4, 2, 5
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    q, k, v, _ = make(total, h, hk, d, dtype, 31)
    want = reference(q, k, v, cu)[0]
    {"q": q, "k": k, "v": v}[place][at, 1, col] = float(fill)
    bad = poisoned(place, fill, at, 1, col, cu, h, hk, total, d)[0]
    for grad in (False, True):  # with a gradient to come the forward also saves what out's rounding left over
        got = packed_attention(q.requires_grad_(grad), k, v, torch.tensor(cu, dtype=torch.int32, device="cuda")).detach()
        assert not torch.isfinite(got[bad]).any()
        assert err(got[~bad], want[~bad]) <= OUT[dtype] * U[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 36, 128))
@pytest.mark.parametrize("place,fill", (("q", "nan"), ("k", "nan"), ("v", "nan"), ("v", "inf"), ("v", "-inf"),
                                        ("do", "nan"), ("do", "inf")))
@pytest.mark.parametrize("lengths,at,total", NAN_LENGTHS)
@pytest.mark.parametrize("h,hk", ((4, 2), (16, 2)))
def test_non_finite_values_reach_the_gradients_that_meet_them_only(dtype, d, place, fill, lengths, at, total, h, hk):
    """The same of dq, dk and dv, with the heads of a group in one block and shared out over several."""
    col = 5
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    q, k, v, do = make(total, h, hk, d, dtype, 31)
    want = reference(q, k, v, cu, do)[1:]
    x = [y.clone() for y in (q, k, v, do)]
    x["qkv".index(place) if place != "do" else 3][at, 1, col] = float(fill)
    reach = poisoned(place, fill, at, 1, col, cu, h, hk, total, d)[1:]
    a, b, c = (y.requires_grad_(True) for y in x[:3])
    out = packed_attention(a, b, c, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    for got, ref, bad in zip(torch.autograd.grad(out, (a, b, c), x[3]), want, reach):
        assert not torch.isfinite(got[bad]).any()
        assert torch.isfinite(got[~bad]).all()
        off = (got[~bad].double() - ref[~bad]).norm().item()
        floor = 2.0 ** -20 * do.double().norm().item() * d ** 0.5
        assert off <= GRAD[dtype] * U[dtype] * ref[~bad].norm().item() + floor


@pytest.mark.parametrize("fill", (float("inf"), -float("inf"), float("nan"), 60000.0))
@pytest.mark.parametrize("place", ("v", "do"))
def test_small_fp16_gradients_beside_a_large_entry(place, fill):
    """dO of size 2^-16 (an unscaled mean over tokens) beside an entry of another sequence that is not finite, or large: dS
    is still held in the range of fp16.  Keys of size 2^8 beside queries of 2^-8 make a dq that fp16 can hold."""
    cu = [0, 256, 700]
    q, k, v, do = make(700, 4, 2, 64, torch.float16, 41)
    q, k, do = q * 2.0 ** -8, k * 2.0 ** 8, do * 2.0 ** -16
    want = reference(q, k, v, cu, do)[1:]
    {"v": v, "do": do}[place][100, 1, 3] = fill
    x = [y.requires_grad_(True) for y in (q, k, v)]
    out = packed_attention(*x, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    for got, ref in zip(torch.autograd.grad(out, x, do), want):
        # the results themselves are fp16: half a step of its smallest numbers, 2^-25, each, beside the relative bound
        off = (got[256:].double() - ref[256:]).norm().item()
        assert off <= GRAD[torch.float16] * U[torch.float16] * ref[256:].norm().item() + 2.0 ** -25 * ref[256:].numel() ** 0.5


def test_everything_not_finite():
    """Inputs of NaN only come back as NaN, and calls after it are as ever."""
    for dtype in DTYPES:
        q, k, v, do = make(2000, 4, 2, 64, dtype, 37)
        cu = torch.tensor([0, 900, 901, 2000], dtype=torch.int32, device="cuda")
        x = [torch.full_like(y, float("nan")).requires_grad_(True) for y in (q, k, v)]
        out = packed_attention(*x, cu)
        assert torch.isnan(out).all()
        assert all(torch.isnan(y).all() for y in torch.autograd.grad(out, x, do))
        check([0, 900, 901, 2000], 4, 2, 64, dtype, seed=37)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Scores of several hundreds: the running maximum moves by more than exp2's range from tile to tile."""
    t, h, d = 520, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    q = (8 * torch.randn(t, h, d, device="cuda", generator=g)).to(dtype)
    k = (8 * torch.randn(t, h, d, device="cuda", generator=g)).to(dtype)
    k = (k.float() * torch.linspace(0.05, 2, t, device="cuda")[:, None, None]).to(dtype)
    v = torch.randn(t, h, d, device="cuda", generator=g).to(dtype)
    ref = reference(q, k, v, [0, t])[0]
    out = packed_attention(q, k, v, torch.tensor([0, t], dtype=torch.int32, device="cuda"))
    # scores up to ~1000 carry 64 rounded products each: their own error, 1000 * 8 * 2^-24, adds to P
    assert err(out, ref) <= OUT[dtype] * U[dtype] + 1000 * 8 * 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 36))
def test_very_large_scores(dtype, d):
    """Scores from 1e8 to 1e11: equal ones share their weight, and one that is far above the rest has all of it.  The
    products of a score are whole multiples of 2^18 whose sums are exact in fp32, so both hold exactly."""
    t, h = 300, 2
    g = torch.Generator(device="cuda").manual_seed(9)
    v = torch.randn(t, h, d, device="cuda", generator=g).to(dtype)
    for size in (3 * 2 ** 10, 5 * 2 ** 11, 3 * 2 ** 13, 7 * 2 ** 13):
        q = torch.full((t, h, d), float(size), device="cuda", dtype=dtype)
        q[::3] = -q[::3]
        cu = torch.tensor([0, 100, t], dtype=torch.int32, device="cuda")
        same = torch.full_like(q, float(size))
        assert err(packed_attention(q, same, v, cu), reference(q, same, v, [0, 100, t])[0]) <= OUT[dtype] * U[dtype]
        one = same / 2
        one[[20, 90, 130, 259]] = same[0]
        assert err(packed_attention(q, one, v, cu), reference(q, one, v, [0, 100, t])[0]) <= OUT[dtype] * U[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", (64, 96, 80))
def test_slices_of_one_projection(dtype, d):
    check([0, 150, 331], 4, 2, d, dtype, fused=True)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_odd_strides(dtype):
    """Heads outside of tokens, a row pitch that is no multiple of 16 bytes, a last dimension that is not contiguous,
    a shifted base, and k / v expanded over heads."""
    t, h, d = 200, 4, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    cu = torch.tensor([0, 77, 200], dtype=torch.int32, device="cuda")
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    wide = r(t * h * (d + 1) + 3)
    makes = {
        "heads outside": lambda: r(h, t, d).transpose(0, 1),
        "odd pitch": lambda: r(t, h, d + 1)[..., :d],
        "last not contiguous": lambda: r(t, d, h).transpose(1, 2),
        "shifted": lambda: wide[3:3 + t * h * d].view(t, h, d),
        "expanded heads": lambda: r(t, 1, d).expand(t, h, d),
        "expanded tokens": lambda: r(1, h, d).expand(t, h, d),
    }
    plain = lambda: r(t, h, d)  # noqa: E731
    for name, f in makes.items():
        for place in range(3):
            x = [plain(), plain(), plain()]
            x[place] = f()
            do = r(t, h, d)
            ref = reference(*x, [0, 77, 200], do)
            y = [a.detach().requires_grad_(True) for a in x]
            out = packed_attention(*y, cu)
            assert err(out, ref[0]) <= OUT[dtype] * U[dtype], (name, place)
            for got, want in zip(torch.autograd.grad(out, y, do), ref[1:]):
                grad_close(got, want, do, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shared_keys_gradient_of_a_broadcast_input(dtype):
    """k and v as an expanded (broadcast) leaf: the gradient sums over the copies."""
    t, h, d = 140, 4, 64
    q, _, _, do = make(t, h, h, d, dtype, 7)
    base = torch.randn(t, 1, d, device="cuda").to(dtype).requires_grad_(True)
    q = q.requires_grad_(True)
    cu = torch.tensor([0, t], dtype=torch.int32, device="cuda")
    out = packed_attention(q, base.expand(t, h, d), base.expand(t, h, d), cu)
    got, = torch.autograd.grad(out, (base,), do)
    _, _, dk, dv = reference(q, base, base, [0, t], do)
    # the copies' gradients are rounded one by one before autograd adds them up
    grad_close(got, dk + dv, do, dtype, times=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l", ((1, 1), (3, 1), (5, 77), (2, 128), (3, 300), (0, 4), (2, 0)))
def test_rows_of_equal_length(dtype, b, l):
    h, hk, d = 4, 2, 96
    q, k, v, do = make(b * l, h, hk, d, dtype, 11)
    ref = reference(q, k, v, [i * l for i in range(b + 1)], do)
    q, k, v = (x.view(b, l, x.shape[1], d).requires_grad_(True) for x in (q, k, v))
    out = packed_attention(q, k, v)
    assert out.shape == (b, l, h, d)
    grads = torch.autograd.grad(out, (q, k, v), do.view(b, l, h, d))
    if b * l == 0:
        return
    assert err(out.flatten(0, 1), ref[0]) <= OUT[dtype] * U[dtype]
    for got, want in zip(grads, ref[1:]):
        grad_close(got.flatten(0, 1), want, do, dtype)


def test_scale():
    check([0, 100, 190], 2, 2, 64, torch.bfloat16, scale=0.5)
    check([0, 100, 190], 2, 2, 64, torch.float32, scale=0.01)


@pytest.mark.parametrize("which", (0, 1, 2))
def test_gradient_against_differences(which):
    """Central differences of the kernel's own forward in fp32 along a direction: the step h = 2^-6 leaves
    h^2 |f'''| / 6 < 1e-4 of the scale of f and 2^-24 |f| / h < 1e-4 of rounding."""
    t, h, hk, d = 90, 2, 1, 32
    q, k, v, do = make(t, h, hk, d, torch.float32, 13)
    cu = torch.tensor([0, 33, 90], dtype=torch.int32, device="cuda")
    x = [a.detach().requires_grad_(True) for a in (q, k, v)]
    g = torch.autograd.grad(packed_attention(*x, cu), x, do)[which]
    u = torch.randn_like(x[which])
    f = lambda y: (packed_attention(*[y if i == which else a.detach() for i, a in enumerate(x)], cu).double()  # noqa: E731
                   * do.double()).sum().item()
    step = 2.0 ** -6
    diff = (f(x[which].detach() + step * u) - f(x[which].detach() - step * u)) / (2 * step)
    want = (g.double() * u.double()).sum().item()
    assert abs(diff - want) <= 2e-3 * (g.double().norm() * u.double().norm()).item()


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeatable(dtype):
    q, k, v, do = make(700, 8, 4, 96, dtype, 17)
    cu = torch.tensor([0, 3, 400, 700], dtype=torch.int32, device="cuda")
    x = [a.detach().requires_grad_(True) for a in (q, k, v)]
    runs = []
    for _ in range(3):
        out = packed_attention(*x, cu)
        runs.append((out.detach(), *torch.autograd.grad(out, x, do)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_another_stream_and_no_wait():
    """The work goes to the caller's current stream, forward and backward."""
    q, k, v, do = make(400, 4, 2, 64, torch.bfloat16, 19)
    cu = torch.tensor([0, 400], dtype=torch.int32, device="cuda")
    ref = reference(q, k, v, [0, 400], do)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = [a.detach().clone().requires_grad_(True) for a in (q, k, v)]
        out = packed_attention(*x, cu)
        grads = torch.autograd.grad(out, x, do)
    s.synchronize()
    assert err(out, ref[0]) <= OUT[torch.bfloat16] * U[torch.bfloat16]
    for got, want in zip(grads, ref[1:]):
        assert err(got, want) <= GRAD[torch.bfloat16] * U[torch.bfloat16]


def test_in_a_cuda_graph():
    q, k, v, _ = make(300, 4, 2, 96, torch.bfloat16, 23)
    cu = torch.tensor([0, 120, 300], dtype=torch.int32, device="cuda")
    want = packed_attention(q, k, v, cu)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = packed_attention(q, k, v, cu)
    new = torch.tensor([0, 7, 300], dtype=torch.int32, device="cuda")
    g.replay()
    assert torch.equal(out, want)
    cu.copy_(new)  # other lengths under the same graph: the offsets are read on the device
    g.replay()
    assert torch.equal(out, packed_attention(q, k, v, new))


def test_refusals():
    q, k, v, _ = make(10, 4, 2, 64, torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError):
        packed_attention(q, k.float(), v, cu)
    with pytest.raises(TypeError):
        packed_attention(q.double(), k.double(), v.double(), cu)
    with pytest.raises(RuntimeError):
        packed_attention(q.cpu(), k.cpu(), v.cpu(), cu.cpu())
    with pytest.raises(RuntimeError):
        packed_attention(q, k, v, cu.cpu())
    for bad in (cu.long(), cu[:1], cu.view(1, 2)):
        with pytest.raises(ValueError):
            packed_attention(q, k, v, bad)
    with pytest.raises(ValueError):
        packed_attention(q, k, v)           # 3-D without offsets
    with pytest.raises(ValueError):
        packed_attention(q[:, :3], k, v, cu)  # 3 heads over 2
    with pytest.raises(ValueError):
        packed_attention(q, k[:9], v[:9], cu)
    with pytest.raises(ValueError):
        packed_attention(q, k, v[..., :32], cu)
    with pytest.raises(ValueError):
        packed_attention(*make(4, 1, 1, 136, torch.bfloat16)[:3], torch.tensor([0, 4], dtype=torch.int32, device="cuda"))
    for s in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            packed_attention(q, k, v, cu, s)
