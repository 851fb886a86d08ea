"""Rotary positions against their definition in 64 bits: types, both pairings, parts of a head, odd sizes, strides, far
positions, gradients against the formula's and against differences.

Tolerances.  u = 2^-24 (fp32), 2^-11 (fp16), 2^-8 (bf16).  A pair (a, b) of norm r turns into one of norm r, so errors
are measured against r times the gain.  In fp32: the rest of an angle, below pi / 4, is rounded twice (conversion and
factor: 2 * 0.79 u), its series add about 2 u each, cos or sin times the gain one, two products and a sum 2 u: under 8 u.
16-bit results add one rounding of the value itself.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from model.mhc_rotary import Rotary, rotate

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(rotary, x, positions, sign=1.0):
    """Every pair as a complex number times gain e^(i position frequency), in fp64; and the pairs' norms."""
    n = rotary.dim
    y = x.detach().double().clone()
    w = rotary.inv_freq.to(x.device)
    a = positions.double()[..., None] * w * sign
    turn = torch.complex(a.cos(), a.sin())[..., None, :] * rotary.gain
    size = torch.zeros_like(y)
    if rotary.interleaved:
        z = torch.view_as_complex(y[..., :n].unflatten(-1, (-1, 2)).contiguous())
        size[..., :n] = (z.abs() * rotary.gain).repeat_interleave(2, -1)
        y[..., :n] = torch.view_as_real(z * turn).flatten(-2)
    else:
        z = torch.complex(y[..., :n // 2].contiguous(), y[..., n // 2:n].contiguous())
        size[..., :n] = (z.abs() * rotary.gain).repeat(*[1] * (z.dim() - 1), 2)
        z = z * turn
        y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
    return y, size


def check(got, rotary, x, positions, sign=1.0):
    want, size = reference(rotary, x, positions, sign)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    bound = 8 * U[torch.float32] * size
    if x.dtype != torch.float32:
        # one rounding of the value that fp32 gives; below the type's normal range half its smallest step
        tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
        bound = bound + U[x.dtype] * (want.abs() + bound) + tiny
        bound[..., rotary.dim:] = 0
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off - bound).max().item()
    assert torch.equal(got[..., rotary.dim:], x[..., rotary.dim:])


@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("d,part", ((96, 96), (96, 32), (128, 42), (40, 20), (64, 8), (2, 2), (7, 4), (256, 256), (256, 2), (33, 32)))
@pytest.mark.parametrize("dtype", tuple(U))
def test_forward(dtype, d, part, interleaved):
    torch.manual_seed(d + part)
    rotary = Rotary(part, 1e6 if part > 2 else 100.0, interleaved=interleaved, gain=1.25)
    q, k = torch.randn(61, 5, d, device="cuda", dtype=dtype), torch.randn(61, 2, d, device="cuda", dtype=dtype)
    pos = torch.randint(0, 5000, (61,), device="cuda")
    for p in (pos, pos.int(), None):
        a, b = rotate(rotary, q, k, p)
        at = torch.arange(61, device="cuda") if p is None else p
        check(a, rotary, q, at)
        check(b, rotary, k, at)


@pytest.mark.parametrize("t,h,hk", ((1, 1, 1), (1, 8, 4), (3, 3, 1), (17, 16, 16), (2049, 8, 4), (5, 200, 3)))
def test_tokens_and_heads(t, h, hk):
    rotary = Rotary(64)
    q, k = torch.randn(t, h, 80, device="cuda").bfloat16(), torch.randn(t, hk, 80, device="cuda").bfloat16()
    a, b = rotate(rotary, q, k)
    at = torch.arange(t, device="cuda")
    check(a, rotary, q, at)
    check(b, rotary, k, at)


def test_rows():
    """(B, L, heads, D): positions from 0 in every row, for every row alike, for every token."""
    rotary = Rotary(32, interleaved=True)
    q, k = torch.randn(3, 50, 4, 48, device="cuda"), torch.randn(3, 50, 2, 48, device="cuda")
    at = torch.arange(50, device="cuda")
    far = torch.randint(0, 100000, (3, 50), device="cuda")
    for p, want in ((None, at.expand(3, 50)), (at + 7, (at + 7).expand(3, 50)), (far, far), (far.int(), far)):
        a, b = rotate(rotary, q, k, p)
        check(a, rotary, q, want)
        check(b, rotary, k, want)


def test_strides():
    rotary = Rotary(64)
    at = torch.arange(40, device="cuda")
    qkv = torch.randn(40, 12, 64, device="cuda").bfloat16()
    q, k, _ = qkv.split((8, 2, 2), 1)
    a, b = rotate(rotary, q, k)
    check(a, rotary, q, at)
    check(b, rotary, k, at)
    # rows that begin at no multiple of 16 bytes, heads before tokens, every other element, one row for all
    buf = torch.randn(40 * 8 * 64 + 3, device="cuda").half()
    for q in (buf[3:].view(40, 8, 64), buf[1:-2].view(40, 8, 64), torch.randn(8, 40, 64, device="cuda").half().transpose(0, 1),
              torch.randn(40, 8, 128, device="cuda").half()[..., ::2], torch.randn(1, 8, 64, device="cuda").half().expand(40, 8, 64),
              torch.randn(40, 1, 64, device="cuda").half().expand(40, 8, 64)):
        a, b = rotate(rotary, q, q[:, :1])
        check(a, rotary, q, at)
        check(b, rotary, q[:, :1], at)


def test_far_positions():
    """Frequencies that are powers of two, so that fp64 holds the angles: positions up to 2^40, and negative ones."""
    rotary = Rotary(16, inv_freq=[2.0 ** -i for i in range(8)])
    pos = torch.tensor([0, 1, -1, 12345, 2 ** 31 - 1, -2 ** 31, 2 ** 33 + 5, 2 ** 40 + 12345, -2 ** 40 - 1], device="cuda")
    q = torch.randn(9, 4, 16, device="cuda")
    a, b = rotate(rotary, q, q[:, :2], pos)
    check(a, rotary, q, pos)
    check(b, rotary, q[:, :2], pos)
    small = pos[:6].int()
    check(rotate(rotary, q[:6], q[:6, :1], small)[0], rotary, q[:6], small)


def test_scaled():
    """By parts, beyond the trained length, and plainly stretched."""
    pos = torch.randint(0, 40000, (33,), device="cuda")
    q = torch.randn(33, 4, 96, device="cuda")
    for rotary in (Rotary(96, 1e6, factor=16, original_length=2048), Rotary(96, 1e6, factor=4.0),
                   Rotary(96, 1e6, factor=16, original_length=2048, gain=1.0)):
        check(rotate(rotary, q, q, pos)[0], rotary, q, pos)


@pytest.mark.parametrize("dtype", tuple(U))
@pytest.mark.parametrize("interleaved,d,part", ((False, 96, 96), (True, 80, 40), (False, 42, 42)))
def test_gradients(dtype, interleaved, d, part):
    rotary = Rotary(part, interleaved=interleaved, gain=1.1)
    q = torch.randn(2, 37, 6, d, device="cuda", dtype=dtype).requires_grad_(True)
    k = torch.randn(2, 37, 2, d, device="cuda", dtype=dtype).requires_grad_(True)
    at = torch.arange(37, device="cuda").expand(2, 37)
    a, b = rotate(rotary, q, k)
    # gradients that come at strides of their own
    ga = torch.randn(2, 6, 37, d, device="cuda", dtype=dtype).transpose(1, 2)
    gb = torch.randn(2, 37, 2, d, device="cuda", dtype=dtype)
    da, db = torch.autograd.grad((a, b), (q, k), (ga, gb), retain_graph=True)
    check(da, rotary, ga, at, -1.0)
    check(db, rotary, gb, at, -1.0)
    # asked for one of them; with one of the outputs unused
    assert torch.equal(torch.autograd.grad(a, q, ga, retain_graph=True)[0], da)
    assert torch.equal(torch.autograd.grad((a, b), k, (ga, gb))[0], db)


def test_gradient_against_differences():
    """The map is linear: a difference of any size is exact but for fp32's roundings, 8 u of the pairs' norms each way."""
    rotary = Rotary(24, interleaved=True)
    q = torch.randn(20, 3, 32, device="cuda").requires_grad_(True)
    g, step = torch.randn(20, 3, 32, device="cuda"), torch.randn(20, 3, 32, device="cuda")
    a, _ = rotate(rotary, q, q.detach())
    grad, = torch.autograd.grad(a, q, g)
    with torch.no_grad():
        hi, lo = (rotate(rotary, q + s * step, q)[0].double() for s in (0.5, -0.5))
    slope = ((hi - lo) * g.double()).sum().item()
    size = (g.double().abs() * (q.double().abs() + step.double().abs())).sum().item() * math.sqrt(2)
    assert abs(slope - (grad.double() * step.double()).sum().item()) < 32 * U[torch.float32] * size


def test_frozen_and_refused():
    rotary = Rotary(32)
    q, k = torch.randn(9, 4, 32, device="cuda", requires_grad=True), torch.randn(9, 4, 32, device="cuda")
    a, b = rotate(rotary, q, k)
    assert a.requires_grad and not torch.autograd.grad(a.sum(), q, create_graph=False)[0].requires_grad
    a, b = rotate(rotary, q, k)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(a.square().sum(), q, create_graph=True)
    with torch.no_grad():
        assert not rotate(rotary, q, k)[0].requires_grad
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        rotate(rotary, fwad.make_dual(k, torch.ones_like(k)), k)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: rotate(rotary, x, x)[0], (k,), check_trace=False)
    for bad in (lambda: rotate(rotary, q, k.half()), lambda: rotate(rotary, q.long(), k.long()),
                lambda: rotate(rotary, q, k, torch.zeros(9, device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: rotate(rotary, q[:8], k), lambda: rotate(rotary, q[..., :30], k[..., :30]), lambda: rotate(rotary, q[0], k[0]),
                lambda: rotate(rotary, q, k, torch.zeros(8, dtype=torch.int64, device="cuda")),
                lambda: rotate(rotary, q, k, torch.zeros(1, 9, dtype=torch.int64, device="cuda")),
                lambda: rotate(Rotary(2), torch.randn(4, 2, 300, device="cuda"), torch.randn(4, 2, 300, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        rotate(rotary, q.cpu(), k.cpu())
    with pytest.raises(RuntimeError, match="CUDA"):
        rotate(rotary, q, k, torch.zeros(9, dtype=torch.int64))


def test_empty():
    rotary = Rotary(32)
    q = torch.randn(0, 4, 32, device="cuda", requires_grad=True)
    a, b = rotate(rotary, q, torch.randn(0, 2, 32, device="cuda"))
    assert a.shape == (0, 4, 32) and torch.autograd.grad(a.sum(), q)[0].shape == (0, 4, 32)
    assert rotate(rotary, torch.randn(2, 0, 4, 32, device="cuda"), torch.randn(2, 0, 2, 32, device="cuda"))[0].shape == (2, 0, 4, 32)


def test_special_values():
    """A NaN or an infinity reaches its own pair only."""
    rotary = Rotary(32)
    q = torch.randn(4, 2, 32, device="cuda")
    clean = rotate(rotary, q, q)[0]
    q[1, 0, 3], q[2, 1, 20] = math.nan, math.inf
    a = rotate(rotary, q, q)[0]
    hit = torch.zeros_like(a, dtype=torch.bool)
    hit[1, 0, [3, 19]] = hit[2, 1, [4, 20]] = True
    assert torch.equal(a[~hit], clean[~hit]) and not torch.isfinite(a[hit]).any()


def test_captured():
    """Forward and backward in one graph, replayed with other positions; an eager graph of other leaves in between."""
    rotary = Rotary(64)
    q, k = torch.randn(33, 4, 64, device="cuda").bfloat16().requires_grad_(True), torch.randn(33, 2, 64, device="cuda").bfloat16()
    g, pos = torch.randn(33, 4, 64, device="cuda").bfloat16(), torch.arange(33, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(rotate(rotary, q, k, pos)[0], q, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = rotate(rotary, q, k, pos)
        d, = torch.autograd.grad(a, q, g)
    for shift in (0, 1000):
        pos.copy_(torch.arange(33, device="cuda") + shift)
        graph.replay()
        check(a.detach(), rotary, q, pos)
        check(b, rotary, k, pos)
        check(d, rotary, g, pos, -1.0)


def test_side_stream_and_repeatable():
    rotary = Rotary(96)
    q, k = torch.randn(4000, 8, 96, device="cuda").bfloat16(), torch.randn(4000, 4, 96, device="cuda").bfloat16()
    want = rotate(rotary, q, k)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotate(rotary, q, k)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_positions_changed_before_the_backward_pass():
    rotary = Rotary(32)
    pos = torch.arange(8, device="cuda")
    q = torch.randn(8, 2, 32, device="cuda", requires_grad=True)
    a, _ = rotate(rotary, q, q.detach(), pos)
    pos += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        a.sum().backward()


def test_made_in_inference_mode():
    with torch.inference_mode():
        rotary = Rotary(32)
        q = torch.randn(9, 4, 32, device="cuda")
        check(rotate(rotary, q, q)[0], rotary, q, torch.arange(9, device="cuda"))
    q = torch.randn(9, 4, 32, device="cuda", requires_grad=True)
    g = torch.randn(9, 4, 32, device="cuda")
    d, = torch.autograd.grad(rotate(rotary, q, q.detach())[0], q, g)
    check(d, rotary, g, torch.arange(9, device="cuda"), -1.0)


def test_what_is_frozen_wants_no_gradient():
    """As with torch's operators: the turned keys of frozen keys are no part of the graph, so that attention behind them
    computes no gradient for them and a cache takes them."""
    rotary = Rotary(32)
    q, k = torch.randn(9, 4, 32, device="cuda"), torch.randn(9, 2, 32, device="cuda")
    g = torch.randn(9, 4, 32, device="cuda")
    at = torch.arange(9, device="cuda")
    a, b = rotate(rotary, q.clone().requires_grad_(True), k)
    assert a.requires_grad and not b.requires_grad and b.grad_fn is None
    check(b, rotary, k, at)
    leaf = k.clone().requires_grad_(True)
    a, b = rotate(rotary, q, leaf)
    assert b.requires_grad and not a.requires_grad
    check(a, rotary, q, at)
    check(torch.autograd.grad(b, leaf, g[:, :2])[0], rotary, g[:, :2], at, -1.0)
    leaf = q.clone().requires_grad_(True)
    both = rotate(rotary, leaf, leaf)
    assert all(x.requires_grad for x in both)
    d, = torch.autograd.grad(both, leaf, (g, g))
    want = reference(rotary, g, at, -1.0)[0] * 2
    assert (d.double() - want).abs().max() <= 32 * U[torch.float32] * 2 * g.abs().max().item() * math.sqrt(2)
