"""Host-side checks of the operators of answering: bad arguments come back as status codes before any CUDA call, the
Python entry points refuse what the kernels do not take, frequencies in fixed point against exact arithmetic, masks of
trees.  Nothing is launched."""

import ctypes
import os
from fractions import Fraction

import pytest
import torch

P = ctypes.c_void_p(4096)      # never dereferenced
ODD = ctypes.c_void_p(4097)
FOUR = (ctypes.c_int64 * 4)(512, 64, 256, 64)
SIX = (ctypes.c_int64 * 6)(512, 64, 256, 64, 256, 64)
TWO = (ctypes.c_int64 * 2)(512, 64)


class RotaryArg(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_void_p), ("part", ctypes.c_int32), ("interleaved", ctypes.c_int32), ("gain", ctypes.c_float)]


class Cache(ctypes.Structure):
    _fields_ = [("keys", ctypes.c_void_p), ("values", ctypes.c_void_p), ("pages", ctypes.c_int64), ("strides", ctypes.c_int64 * 8),
                ("dtype", ctypes.c_int32), ("layers", ctypes.c_int32), ("page_size", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("dim", ctypes.c_int32)]


class Step(ctypes.Structure):
    _fields_ = [("page_table", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("cu_tokens", ctypes.c_void_p), ("table_pitch", ctypes.c_int64),
                ("T", ctypes.c_int64), ("table_width", ctypes.c_int32), ("batch", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    from model import _native
    if not os.path.exists(_native.LIB_PATH) or not os.path.exists(_native.HOST_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _native.load_library()


def rot(part=64, turns=4096):
    return RotaryArg(turns, part, 0, 1.0)


def cache(**kw):
    a = dict(keys=4096, values=4096, pages=10, dtype=1, layers=1, page_size=16, kv_heads=4, dim=64) | kw
    c = Cache(strides=(ctypes.c_int64 * 8)(0, 4096, 256, 64, 0, 4096, 256, 64))
    for k, v in a.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def step(**kw):
    a = dict(page_table=4096, lengths=4096, cu_tokens=4096, table_pitch=8, T=20, table_width=8, batch=3) | kw
    s = Step()
    for k, v in a.items():
        setattr(s, k, v)
    return ctypes.byref(s)


def rotate(lib, r=None, q=P, qo=P, H=8, k=P, ko=P, Hk=4, dtype=1, T=10, D=64, strides=FOUR, pos=None, pb=0, period=0):
    return lib.mhc_rotate(ctypes.byref(r or rot()), q, qo, H, k, ko, Hk, dtype, T, D, strides, pos, pb, period, 0, None)


def test_rotate_refusals(lib):
    assert rotate(lib, T=0) == 0
    assert lib.mhc_rotate(None, P, P, 8, P, P, 4, 1, 10, 64, FOUR, None, 0, 0, 0, None) == -1
    assert rotate(lib, dtype=5) == -2 and rotate(lib, pos=P, pb=2) == -2
    assert rotate(lib, D=257) == -3 and rotate(lib, T=-1) == -3 and rotate(lib, H=0, Hk=0) == -3 and rotate(lib, period=-1) == -3
    for part in (0, 3, 66, -2):
        assert rotate(lib, r=rot(part)) == -3 and b"even part" in lib.mhc_last_error()
    assert rotate(lib, r=rot(turns=0)) == -1 and rotate(lib, r=rot(turns=4100)) == -4
    assert rotate(lib, q=None) == -1 and rotate(lib, ko=None) == -1 and rotate(lib, strides=None) == -1
    assert rotate(lib, q=ODD) == -4 and rotate(lib, pos=ODD, pb=4) == -4


def append(lib, c=None, s=None, k=P, v=P, q=P, qo=P, H=8, strides=SIX, r=None, pos=None, pb=0):
    return lib.mhc_append_kv(c or cache(), s or step(), k, v, q, qo, H, strides, ctypes.byref(r) if r else None, pos, pb, None)


def test_append_refusals(lib):
    assert append(lib, s=step(T=0)) == 0
    assert append(lib, c=cache(dtype=3)) == -2
    for kw in (dict(pages=-1), dict(page_size=0), dict(kv_heads=0), dict(dim=0), dict(dim=257)):
        assert append(lib, c=cache(**kw)) == -3
    for kw in (dict(T=-1), dict(batch=-1), dict(table_width=-1), dict(table_width=1 << 30)):
        assert append(lib, s=step(**kw)) == -3
    for kw in (dict(lengths=None), dict(cu_tokens=None), dict(page_table=None)):
        assert append(lib, s=step(**kw)) == -1
    assert append(lib, c=cache(keys=None)) == -1 and append(lib, k=None) == -1 and append(lib, strides=None) == -1
    assert append(lib, c=cache(keys=4097)) == -4 and append(lib, s=step(lengths=4098)) == -4 and append(lib, v=ODD) == -4
    assert append(lib, r=rot(66)) == -3 and append(lib, r=rot(), q=None) == -1
    assert lib.mhc_append_kv(None, step(), P, P, P, P, 8, SIX, None, None, 0, None) == -1


def test_keep_refusals(lib):
    assert lib.mhc_keep_drafts(cache(layers=0), step(), P, P, None) == 0
    assert lib.mhc_keep_drafts(cache(), step(batch=0), P, P, None) == 0
    assert lib.mhc_keep_drafts(cache(), step(), None, P, None) == -1
    assert lib.mhc_keep_drafts(cache(), step(), P, ODD, None) == -4
    assert lib.mhc_keep_drafts(cache(layers=70000), step(), P, P, None) == -3


def attend(lib, c=None, s=None, q=P, H=8, strides=TWO, mask=None, scale=0.1, out=P, ws=P, n=1 << 30):
    return lib.mhc_cached_attn(c or cache(), s or step(), q, H, strides, mask, scale, out, ws, n, None)


def test_attention_refusals(lib):
    assert attend(lib, s=step(T=0)) == 0
    assert attend(lib, c=cache(dim=160)) == -3 and attend(lib, H=6) == -3 and attend(lib, H=0) == -3
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert attend(lib, scale=scale) == -3
    assert attend(lib, q=None) == -1 and attend(lib, out=None) == -1 and attend(lib, strides=None) == -1
    assert attend(lib, q=ODD) == -4 and attend(lib, mask=ctypes.c_void_p(4100)) == -4
    assert attend(lib, ws=None) == -5 and attend(lib, n=16) == -5 and attend(lib, ws=ctypes.c_void_p(4096 + 16)) == -4
    # more work than the units of one call can count
    assert attend(lib, s=step(T=1 << 30, table_width=1 << 26), n=1 << 40) == -3
    need = lib.mhc_cached_attn_workspace(cache(), step(), 8)
    assert 0 < need < 1 << 28
    assert lib.mhc_cached_attn_workspace(cache(), step(batch=0), 8) == 0 and lib.mhc_cached_attn_workspace(cache(), step(), 7) == 0


def verify(lib, tokens=P, parents=P, cu=P, batch=2, T=10, target=P, ts=50, draft=P, ds=50, dtype=0, V=50, random=P, path=P, kept=P, nxt=P):
    return lib.mhc_verify_drafts(tokens, parents, cu, batch, T, target, ts, draft, ds, dtype, V, random, path, kept, nxt, None)


def test_verify_refusals(lib):
    assert verify(lib, batch=0, T=0) == 0
    assert verify(lib, dtype=8) == -2
    assert verify(lib, V=0) == -3 and verify(lib, T=-1) == -3 and verify(lib, batch=-1) == -3 and verify(lib, ts=49) == -3 and verify(lib, ds=49) == -3
    for kw in ("tokens", "parents", "cu", "target", "random", "path", "kept", "nxt"):
        assert verify(lib, **{kw: None}) == -1
        assert verify(lib, **{kw: ODD}) == -4


def test_python_refusals():
    """Without a device every entry point says so; shapes are checked where tensors can be."""
    from model.mhc_cache import CacheStep, append_kv, cached_attention, keep_drafts
    from model.mhc_rotary import Rotary, rotate
    from model.mhc_verify import verify_drafts
    r = Rotary(32)
    q, k, pool = torch.zeros(3, 4, 32), torch.zeros(3, 2, 32), torch.zeros(4, 8, 2, 32)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    step = CacheStep(i32(1, 4), i32(1), i32(2))
    for bad in (lambda: rotate(r, q, k), lambda: append_kv(pool, pool, step, k, k), lambda: cached_attention(q, pool, pool, step),
                lambda: keep_drafts(pool, pool, step, i32(3), i32(1)),
                lambda: verify_drafts(torch.zeros(3, dtype=torch.int64), i32(3), i32(2), torch.zeros(3, 9), None, torch.zeros(3))):
        with pytest.raises(RuntimeError, match="CUDA"):
            bad()
    for bad in (lambda: Rotary(3), lambda: Rotary(0), lambda: Rotary(8, theta=-1.0), lambda: Rotary(8, theta=1.0), lambda: Rotary(8, factor=0.5),
                lambda: Rotary(8, factor=2, original_length=0), lambda: Rotary(8, inv_freq=[1.0]), lambda: Rotary(8, inv_freq=[1.0, 2.0, float("inf"), 0.0]),
                lambda: Rotary(8, gain=float("nan")), lambda: Rotary(8, factor=2, original_length=100, slow=0.0)):
        with pytest.raises(ValueError):
            bad()


def test_frequencies_in_fixed_point():
    """turns[i] is frequency / (2 pi) in 2^-64ths, to half of one: pi from Machin's formula in exact fractions."""
    from model.mhc_rotary import Rotary
    def arctan(n):
        return sum(Fraction((-1) ** i, (2 * i + 1) * n ** (2 * i + 1)) for i in range(110))
    pi = 4 * (4 * arctan(5) - arctan(239))
    for r in (Rotary(96, 1e6), Rotary(128, 1e4, factor=8, original_length=4096), Rotary(8, inv_freq=[1.0, 1e-9, 700.25, -0.5])):
        for f, t in zip(r.inv_freq.tolist(), r._host.tolist()):
            exact = Fraction(f) / (2 * pi) * 2 ** 64
            off = (t - exact) % 2 ** 64
            assert min(off, 2 ** 64 - off) <= Fraction(1, 2)


def test_scaled_frequencies():
    """By parts: fast pairs as they were, slow ones divided, a ramp between; the gain."""
    import math

    from model.mhc_rotary import Rotary
    plain, far = Rotary(96, 1e6).inv_freq, Rotary(96, 1e6, factor=16, original_length=2048)
    turns = 2048 * plain / (2 * math.pi)
    assert torch.equal(far.inv_freq[turns > 64], plain[turns > 64])
    assert torch.allclose(far.inv_freq[turns < 0.5], plain[turns < 0.5] / 16, rtol=1e-15, atol=0)
    ratio = far.inv_freq / plain
    assert (ratio[1:] <= ratio[:-1] + 1e-15).all()
    assert far.gain == 0.1 * math.log(16) + 1 and Rotary(96, factor=4).gain == 1.0
    assert torch.allclose(Rotary(96, 1e6, factor=4).inv_freq, plain / 4, rtol=1e-15, atol=0)
    assert Rotary(96, 1e6, factor=16, original_length=2048, gain=1.0).gain == 1.0


def test_tree_mask():
    from model.mhc_cache import tree_mask
    parents = torch.tensor([-1, 0, 0, 1, 3, -1, -1, 0, 1], dtype=torch.int32)
    mask, depth = tree_mask(parents, torch.tensor([0, 5, 6, 6, 9], dtype=torch.int32))
    assert mask.tolist() == [1, 3, 5, 11, 27, 1, 1, 3, 7] and depth.tolist() == [0, 1, 1, 2, 3, 0, 0, 1, 2]
    # rows of no sequence, parents that do not come before their row
    parents = torch.tensor([7, -1, 0, 5, 1, 2 ** 31 - 1, 1, -9], dtype=torch.int32)
    mask, depth = tree_mask(parents, torch.tensor([1, 5], dtype=torch.int32))
    assert mask[1:5].tolist() == [1, 3, 4, 11] and depth.tolist()[:5] == [0, 0, 1, 0, 2] and depth.tolist()[7] == 0
    assert tree_mask(parents[:0], torch.tensor([0], dtype=torch.int32))[0].numel() == 0


def test_sizes_that_32_bits_do_not_hold(lib):
    """Rows of an item are counted in 32 bits, and so are sequences and heads: what they do not hold is refused, where every
    other limit of the call would let it pass."""
    small = dict(kv_heads=1, dim=8)
    for tokens, heads in ((1 << 27, 32), (1 << 26, 32), (1 << 20, 1 << 12)):
        assert attend(lib, c=cache(**small), s=step(T=tokens, table_width=4), H=heads, n=1 << 50) == -3
        assert b"rows" in lib.mhc_last_error()
    wide = cache(kv_heads=16385)
    assert append(lib, c=wide) == -3 and attend(lib, c=wide, H=16385, n=1 << 50) == -3 and lib.mhc_keep_drafts(wide, step(), P, P, None) == -3
    many = step(batch=(1 << 30) + 1)
    assert append(lib, s=many) == -3 and attend(lib, s=many, n=1 << 50) == -3 and lib.mhc_keep_drafts(cache(), many, P, P, None) == -3


def test_tree_mask_of_rows_of_no_sequence():
    """They are first ones, whatever their parents look like; offsets that are none index nothing."""
    from model.mhc_cache import tree_mask
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    mask, depth = tree_mask(i32(-1, 0, 1, 0, 1, 2), i32(0, 3))
    assert mask.tolist() == [1, 3, 7, 1, 1, 1] and depth.tolist() == [0, 1, 2, 0, 0, 0]
    mask, depth = tree_mask(i32(0, 0, -1, 0, 1, 0, 2), i32(2, 2, 4, 4))
    assert mask.tolist() == [1, 1, 1, 3, 1, 1, 1] and depth.tolist() == [0, 0, 0, 1, 0, 0, 0]
    mask, depth = tree_mask(i32(0, 0, 1), i32(0))
    assert mask.tolist() == [1, 1, 1] and depth.tolist() == [0, 0, 0]
    for cu in (i32(-2 ** 31, 2 ** 31 - 1), i32(-9, -5, 2), i32(2 ** 31 - 1, -7, 3), i32(5, 1, 0)):
        mask, depth = tree_mask(i32(0, 1, 2, 0), cu)
        assert mask.shape == depth.shape == (4,) and (depth >= 0).all() and (depth < 4).all()
    for bad in (lambda: tree_mask(i32(-1, 0), i32()), lambda: tree_mask(i32(-1, 0)[None], i32(0, 2)), lambda: tree_mask(i32(-1, 0), i32(0, 2)[None])):
        with pytest.raises(ValueError):
            bad()


def test_frequencies_made_in_inference_mode():
    """An evaluation that is a rotation's first use leaves frequencies that a training step can keep for its backward pass."""
    from model.mhc_rotary import Rotary
    outside = Rotary(16, device="cpu")
    with torch.inference_mode():
        inside = Rotary(16, device="cpu")
        late = outside.turns("meta")
    for x in (inside.turns("cpu"), inside._host, inside.inv_freq, late):
        assert not x.is_inference()
    assert torch.equal(inside.turns("cpu"), outside.turns("cpu"))


@pytest.mark.parametrize("device", ("meta", "cpu"))
def test_frequencies_under_another_default_device(device):
    """A model whose parameters are laid out later is built under a default device that holds no values."""
    from model.mhc_rotary import Rotary
    with torch.device(device):
        r = Rotary(16, device="cpu")
    assert r._host.device.type == r.inv_freq.device.type == "cpu"
    assert torch.equal(r.turns("cpu"), Rotary(16, device="cpu").turns("cpu"))


@pytest.mark.parametrize("dim,theta,factor,length,fast,slow", ((96, 1e6, 16.0, 2048, 32.0, 1.0), (128, 1e4, 4.0, 4096, 32.0, 1.0), (64, 1e6, 8.0, 512, 4.0, 0.5)))
def test_scaled_tables(dim, theta, factor, length, fast, slow):
    """Pair by pair, and the tables that a model with an attention factor of 1, or of its own, multiplies with: pair i turns
    length theta^(-2i/dim) / 2 pi times within the trained length; the pairs at which that is `fast` and `slow`, rounded
    outwards, are the ramp's ends."""
    import math

    from model.mhc_rotary import Rotary
    lo = max(math.floor(dim / 2 * math.log(length / (2 * math.pi * fast), theta)), 0)
    hi = min(math.ceil(dim / 2 * math.log(length / (2 * math.pi * slow), theta)), dim // 2 - 1)
    assert 0 <= lo < hi
    position = torch.arange(0, 4 * length, 97, dtype=torch.float64)[:, None]
    for gain in (1.0, 1.5):
        r = Rotary(dim, theta, factor=factor, original_length=length, fast=fast, slow=slow, gain=gain)
        assert r.gain == gain
        want = []
        for i in range(dim // 2):
            f = theta ** (-2 * i / dim)
            part = 0.0 if i <= lo else 1.0 if i >= hi else (i - lo) / (hi - lo)
            want.append(f * (1 - part) + f / factor * part)
        want = torch.tensor(want, dtype=torch.float64)
        assert torch.allclose(r.inv_freq, want, rtol=1e-14, atol=0)
        # angles up to 4 length, off by 1e-14 of themselves
        assert torch.allclose((position * r.inv_freq).cos() * r.gain, (position * want).cos() * gain, rtol=0, atol=4 * length * 1e-14 * gain + 1e-15)
    assert Rotary(dim, theta, factor=1.0, original_length=length).gain == 1.0
