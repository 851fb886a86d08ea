"""Top-k router against its definition in 64 bits.

Tolerances: fp32 arithmetic on at most E = 512 values a row, an exp of 2 ulp, one division: 32 * 2^-24 relative to
the largest exact value of the tensor for weights and loss; a gradient is a difference of two such products, 128 *
2^-24 of the largest, plus the rounding of its own type.  Indices and counts are equal."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from model.mhc_router import route_topk

EPS = 2.0 ** -24
ROUND = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def reference(z, k, coef, dw, dloss):
    z = z.detach().double().requires_grad_(True)
    t, e = z.shape
    p = z.softmax(-1)
    idx = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
    top = p.gather(1, idx)
    w = top / (top.sum(-1, keepdim=True) + 1e-20)
    counts = torch.zeros(e, dtype=torch.long, device=z.device).index_add_(
        0, idx.flatten(), torch.ones(t * k, dtype=torch.long, device=z.device))
    loss = coef * e * (counts.double() / t * p.mean(0)).sum()
    dz, = torch.autograd.grad((w, loss), (z,), (dw.double(), dloss.double()))
    return w.detach(), idx, counts, loss.detach(), dz


def close(got, want, tol):
    assert torch.isfinite(got).all()
    assert (got.double() - want).abs().max() <= tol * max(want.abs().max().item(), 1e-30)


def check(t, e, k, dtype, logits=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = (torch.randn(t, e, device="cuda", generator=g) * 2).to(dtype) if logits is None else logits
    dw = torch.randn(t, k, device="cuda", generator=g)
    dl = torch.randn((), device="cuda", generator=g)
    ref = reference(z, k, 0.3, dw, dl)
    z = z.detach().requires_grad_(True)
    w, idx, counts, loss = route_topk(z, k, 0.3)
    assert w.dtype == torch.float32 and idx.dtype == torch.int64 and counts.dtype == torch.int64
    assert torch.equal(idx, ref[1]) and torch.equal(counts, ref[2])
    close(w, ref[0], 32 * EPS)
    close(loss, ref[3], 32 * EPS)
    dz, = torch.autograd.grad((w, loss), (z,), (dw, dl))
    assert dz.dtype == z.dtype
    # the weights' part scales with 1 / (sum of the chosen p) and is a difference of like terms
    close(dz, ref[4], 128 * EPS + ROUND[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e,k", ((1, 1), (2, 1), (3, 2), (4, 4), (7, 3), (8, 2), (8, 8), (9, 2), (16, 4), (20, 5),
                                 (31, 31), (32, 8), (60, 6), (64, 6), (64, 64), (100, 1), (128, 8), (160, 6), (256, 8),
                                 (257, 9), (384, 8), (512, 16)))
def test_expert_counts(dtype, e, k):
    check(37, e, k, dtype, seed=e)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t", (1, 2, 31, 255, 256, 257, 1000, 5001, 40000, 200001))
def test_token_counts(dtype, t):
    check(t, 8, 2, dtype, seed=t)
    if t <= 5001:
        check(t, 64, 6, dtype, seed=t + 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_index(dtype):
    z = torch.randint(-2, 3, (500, 24), device="cuda").to(dtype)
    z[z == 0] = -0.0
    z[:, ::3] = z[:, ::3].abs()  # zeros of both signs
    check(500, 24, 5, dtype, z)
    check(50, 8, 3, dtype, torch.zeros(50, 8, device="cuda", dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_experts(dtype):
    """Logits of -inf and of the type's lowest value: such experts have weight 0 and are chosen last."""
    z = torch.randn(64, 16, device="cuda").to(dtype)
    z[:, 5:] = -float("inf")
    check(64, 16, 3, dtype, z.clone())
    z[:, 5:] = torch.finfo(dtype).min
    check(64, 16, 3, dtype, z)
    z = torch.randn(64, 16, device="cuda").to(dtype)
    z[:, 2:] = -float("inf")  # fewer experts than choices
    w, idx, counts, _ = route_topk(z, 4)
    assert (w[:, 2:] == 0).all() and torch.equal(idx[:, 2:], torch.tensor([2, 3], device="cuda").expand(64, 2))
    assert counts[2] == 64 and counts[4:].sum() == 0
    assert torch.allclose(w.sum(-1), torch.ones(64, device="cuda"), atol=4 * EPS)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_without_experts(dtype):
    z = torch.randn(9, 8, device="cuda").to(dtype)
    z[4] = -float("inf")
    z = z.requires_grad_(True)
    w, idx, counts, loss = route_topk(z, 2, 1.0)
    assert (w[4] == 0).all() and idx[4].tolist() == [0, 1] and counts.sum() == 18
    assert torch.isfinite(loss)
    dz, = torch.autograd.grad((w, loss), (z,), (torch.ones_like(w), torch.ones_like(loss)))
    assert torch.isfinite(dz).all() and (dz[4] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_very_large_logits(dtype):
    """Finite rows of any size have a softmax: all alike (a token that no expert may take, masked with the type's
    lowest value or -1e10) 1 / E, one far above the rest 1, and between large logits only their difference counts."""
    lim = torch.finfo(dtype)
    sizes = [lim.min, lim.max, lim.min / 2] + ([] if dtype == torch.float16 else [-1e10, 1e10, -1e11, -1e30, 1e38, 5e9])
    rows = [[s] * 8 for s in sizes]
    rows += [[lim.max] + [0.0] * 7, [0.0] * 5 + [lim.max, lim.min, 1.0], [lim.min] * 7 + [lim.max]]
    if dtype != torch.float16:
        rows += [[3.3e38] + [1.0] * 7, [1e10] + [0.0] * 7, [-1e10] * 7 + [-2e10]]
    if dtype == torch.float32:
        rows += [[1e6 + i for i in range(8)], [-1e7 - i for i in range(8)], [3e9 - 256 * (i % 2) for i in range(8)]]
    z = torch.randn(64, 8, device="cuda").to(dtype)  # ordinary rows beside them
    z[:len(rows)] = torch.tensor(rows, dtype=torch.float64, device="cuda").to(dtype)
    check(64, 8, 3, dtype, z)
    wide = torch.zeros(40, 300, device="cuda", dtype=dtype)
    wide[:20], wide[20:] = lim.min, lim.max
    wide[::2, 7] = 1.0
    check(40, 300, 5, dtype, wide)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_inf_stay_in_their_row(dtype):
    z = torch.randn(300, 8, device="cuda").to(dtype)
    clean = route_topk(z, 2)
    z[7, 3] = float("nan")
    z[9, 4] = -float("nan")
    z[11, 1] = float("inf")
    w, idx, counts, loss = route_topk(z, 2, 1.0)
    assert idx[7, 0] == 3 and idx[9, 0] == 4 and idx[11, 0] == 1
    assert torch.isnan(w[[7, 9, 11]]).any(1).all() and torch.isnan(loss) and counts.sum() == 600
    rest = [i for i in range(300) if i not in (7, 9, 11)]
    assert torch.equal(w[rest], clean.weights[rest]) and torch.equal(idx[rest], clean.experts[rest])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_shapes(dtype):
    base = torch.randn(100, 40, device="cuda").to(dtype)
    for z in (base[:, 3:19], base[:, 8:24], base[::2, :16], base.t()[:16].t(), base[:1].expand(100, 40)[:, :16]):
        check(z.shape[0], 16, 3, dtype, z)
    z = torch.randn(2, 3, 5, 8, device="cuda").to(dtype)
    r = route_topk(z, 2)
    assert r.weights.shape == (2, 3, 5, 2) and r.experts.shape == (2, 3, 5, 2)
    assert torch.equal(r.experts.view(-1, 2), route_topk(z.view(-1, 8), 2).experts)


def test_gradient_against_differences():
    """fp32 logits, a step of 2^-7 along a direction: h^2 of truncation and 2^-24 / h of rounding, both < 1e-3 of the
    gradient's norm.  Logits kept apart so that no choice changes."""
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.stack([torch.randperm(12, device="cuda", generator=g) for _ in range(40)]).float() * 0.3
    u = torch.randn(40, 12, device="cuda", generator=g).clamp(-3, 3)
    dw = torch.randn(40, 3, device="cuda", generator=g)
    x = z.clone().requires_grad_(True)
    w, _, _, loss = route_topk(x, 3, 0.7)
    dz, = torch.autograd.grad((w, loss), (x,), (dw, torch.ones_like(loss)))

    def f(y):
        w, _, _, loss = route_topk(y, 3, 0.7)
        return ((w.double() * dw).sum() + loss.double()).item()

    h = 2.0 ** -7
    diff = (f(z + h * u) - f(z - h * u)) / (2 * h)
    assert abs(diff - (dz.double() * u).sum().item()) <= 2e-3 * (dz.norm() * u.norm()).item()


def test_one_gradient_only():
    z = torch.randn(50, 8, device="cuda")
    zero_w, zero_l = torch.zeros(50, 2, device="cuda"), torch.zeros((), device="cuda")
    dw, dl = torch.randn(50, 2, device="cuda"), torch.ones((), device="cuda")
    for pick in (0, 1):
        x = z.clone().requires_grad_(True)
        w, _, _, loss = route_topk(x, 2, 0.3)
        out, g = ((w,), (dw,)) if pick == 0 else ((loss,), (dl,))
        dz, = torch.autograd.grad(out, (x,), g)
        ref = reference(z, 2, 0.3, dw if pick == 0 else zero_w, dl if pick == 1 else zero_l)
        close(dz, ref[4], 128 * EPS)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("e,k", ((16, 9), (64, 40), (256, 160), (512, 300)))
def test_gradient_of_many_tokens_a_group(dtype, e, k):
    """Three and a half turns of every group of lanes, most experts chosen in one turn and the next, each time by
    another lane: what one turn leaves in shared memory must not meet the next."""
    lanes = min(32, e // 8)
    check(int(3.5 * 8 * torch.cuda.get_device_properties(0).multi_processor_count * (256 // lanes)), e, k, dtype, seed=e)


def test_no_tokens():
    z = torch.empty(0, 8, device="cuda", requires_grad=True)
    w, idx, counts, loss = route_topk(z, 2, 1.0)
    assert w.shape == (0, 2) and idx.shape == (0, 2) and counts.tolist() == [0] * 8 and loss.item() == 0
    dz, = torch.autograd.grad((w, loss), (z,), (torch.ones_like(w), torch.ones_like(loss)))
    assert dz.shape == (0, 8)


def test_repeatable_and_on_another_stream():
    z = torch.randn(30000, 64, device="cuda").bfloat16()
    a = route_topk(z, 6, 1.0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = route_topk(z, 6, 1.0)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals():
    z = torch.randn(4, 8, device="cuda")
    for k in (0, 9, -1):
        with pytest.raises(ValueError):
            route_topk(z, k)
    with pytest.raises(ValueError):
        route_topk(torch.randn(4, 513, device="cuda"), 2)
    with pytest.raises(TypeError):
        route_topk(z.double(), 2)
    with pytest.raises(TypeError):
        route_topk(z.long(), 2)
    with pytest.raises(RuntimeError):
        route_topk(z.cpu(), 2)
