"""The training-step operators together: the benchmark decoder with them against the same decoder on torch's, and the
packed example; the tensor-core attention against the CUDA-core one."""

import os
import sys

import pytest
import torch
import torch.nn.functional as F

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_decoder_with_native_ops_matches_torch_ops(dtype):
    """One step of the MoE + mHC decoder, same weights, same tokens.  fp32: the two differ by fp32 roundings through 2
    layers (1e-4 of the largest gradient).  bf16: the router of torch's side rounds its probabilities to bf16, so a
    token whose choice is a near tie may go to another expert; the losses agree to 2^-8 and the gradients of the
    embedding, which average over the tokens, to 10 %."""
    import bench
    dev = torch.device("cuda")
    args = dict(moe=True, dev=dev, hidden=256, layers=2, heads=4, kv_heads=2, inter=256, vocab=300, dtype=dtype)
    torch.manual_seed(3)
    a = bench._build_decoder(**args)
    b = bench._build_decoder(native_ops=True, **args)
    b.load_state_dict(a.state_dict())
    ids = torch.randint(0, 300, (3, 200), device=dev)
    grads, losses = [], []
    for m in (a, b):
        logits = m(ids)
        loss = F.cross_entropy(logits[:, :-1].reshape(-1, 300).float(), ids[:, 1:].reshape(-1)) + m.aux_loss()
        loss.backward()
        losses.append(loss.item())
        grads.append(m.lm_head.weight.grad.double())
    off = (grads[0] - grads[1]).norm() / grads[0].norm()
    if dtype == torch.float32:
        assert abs(losses[0] - losses[1]) <= 1e-4 * losses[0]
        assert off <= 1e-4
    else:
        assert abs(losses[0] - losses[1]) <= 2.0 ** -8 * losses[0]
        assert off <= 0.1


def test_decoder_has_no_balance_loss_outside_of_training():
    """Evaluation: both sides' auxiliary loss is zero, as in the reference's MoE layer."""
    import bench
    args = dict(moe=True, dev=torch.device("cuda"), hidden=256, layers=2, heads=4, kv_heads=2, inter=256, vocab=300)
    ids = torch.randint(0, 300, (2, 50), device="cuda")
    for native in (False, True):
        torch.manual_seed(3)
        m = bench._build_decoder(native_ops=native, **args)
        m(ids)
        assert m.aux_loss().item() > 0
        m.eval()
        m(ids)
        assert m.aux_loss().item() == 0


@pytest.mark.parametrize("bits", (32, 8))
def test_packed_example_learns(bits):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import train_packed_moe
    losses = train_packed_moe.train(30, bits)
    # a uniform guess over 512 tokens costs log 512 = 6.24
    assert losses[0] > 5.5 and losses[-1] < 0.5 * losses[0]


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_tensor_core_attention_against_cuda_core_attention(dtype):
    """Both from the same inputs; the difference is the tensor-core side's rounding of P and dS (2 u each)."""
    from model import _native as nat
    from model.mhc_attention import packed_attention
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v, do = (torch.randn(1500, h, 96, device="cuda", generator=g).to(dtype) for h in (8, 4, 4, 8))
    cu = torch.tensor([0, 700, 701, 1400], dtype=torch.int32, device="cuda")
    sides = []
    for policy in (nat.PATH_AUTO, nat.PATH_GENERIC):
        prev = nat.lib().mhc_set_path_policy(policy)
        try:
            x = [t.detach().requires_grad_(True) for t in (q, k, v)]
            out = packed_attention(*x, cu)
            sides.append((out.detach(), *torch.autograd.grad(out, x, do)))
        finally:
            nat.lib().mhc_set_path_policy(prev)
    for a, b in zip(*sides):
        assert not torch.equal(a, b)  # two kernels ran
        assert (a.double() - b.double()).norm() <= 4 * u * b.double().norm()


def test_second_derivatives_are_refused():
    from model.mhc_attention import packed_attention
    from model.mhc_router import route_topk
    q = torch.randn(4, 2, 64, device="cuda", requires_grad=True)
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(packed_attention(q, q, q, cu).sum(), q, create_graph=True)
    z = torch.randn(4, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(route_topk(z, 2, 1.0).weights.square().sum(), z, create_graph=True)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor does not require grad: without a check its tangent would be dropped without a word."""
    import torch.autograd.forward_ad as fwad
    from model.mhc_attention import packed_attention
    from model.mhc_router import route_topk
    x = [torch.randn(1, 6, 2, 64, device="cuda") for _ in range(3)]
    z = torch.randn(4, 8, device="cuda")
    with fwad.dual_level():
        for place in range(3):
            for other_grad in (False, True):
                y = [t.clone().requires_grad_(other_grad) for t in x]
                y[place] = fwad.make_dual(x[place], torch.ones_like(x[place]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    packed_attention(*y)
        with pytest.raises(RuntimeError, match="forward-mode"):
            route_topk(fwad.make_dual(z, torch.ones_like(z)), 2, 1.0)
    packed_attention(*x)
    route_topk(z, 2, 1.0)


def test_tracing_is_refused():
    """A trace would keep the empty outputs and not the launch."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from model.mhc_attention import packed_attention
    from model.mhc_router import route_topk
    from model.mhc_adamw import adamw_step

    def step(t):
        adamw_step([t], [t], [t.clone()], [t.square()], step=1, lr=1e-3)
        return t

    q, z = torch.randn(1, 6, 2, 64, device="cuda"), torch.randn(4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(step)(z)
    for grad in (False, True):
        q.requires_grad_(grad)
        z.requires_grad_(grad)
        for f, x in ((lambda t: packed_attention(t, t, t), q), (lambda t: route_topk(t, 2, 1.0).weights, z)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                torch.jit.trace(f, x, check_trace=False)
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(f)(x)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_attention_computes_the_gradients_that_are_asked_for(dtype):
    """Frozen keys and values, or a frozen query: the others' gradients are the same bits as with all three, and those
    not asked for take no memory (counted as the bytes asked of the allocator: what it hands out may be a larger block
    that was free)."""
    from model.mhc_attention import packed_attention
    t, h, hk, d = 6000, 8, 8, 64
    g = torch.Generator(device="cuda").manual_seed(7)
    base = [torch.randn(t, n, d, device="cuda", generator=g).to(dtype) for n in (h, hk, hk)]
    do = torch.randn(t, h, d, device="cuda", generator=g).to(dtype)
    cu = torch.tensor([0, 1000, 1001, 5000], dtype=torch.int32, device="cuda")

    def run(which, leaves):
        x = [b.clone().requires_grad_(i in leaves) for i, b in enumerate(base)]
        out = packed_attention(*x, cu)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_stats()["requested_bytes.all.current"]
        grads = torch.autograd.grad(out, [x[i] for i in which], do)
        return grads, torch.cuda.memory_stats()["requested_bytes.all.peak"] - before

    full, most = run((0, 1, 2), (0, 1, 2))
    size = base[0].numel() * base[0].element_size()
    for which, saved in (((0,), 2), ((1, 2), 1), ((1,), 1), ((2,), 1), ((0, 2), 0)):
        for leaves in (which, (0, 1, 2)):
            grads, peak = run(which, leaves)
            assert all(torch.equal(a, full[i]) for a, i in zip(grads, which))
            assert peak <= most - saved * size


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_attention_gradient_at_an_odd_address(dtype):
    """dO that begins at no multiple of 16 bytes goes through the same kernels as one that does."""
    from model.mhc_attention import packed_attention
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (torch.randn(1, 500, n, 64, device="cuda", generator=g).to(dtype).requires_grad_(True) for n in (4, 2, 2))
    flat = torch.randn(500 * 4 * 64 + 3, device="cuda", generator=g).to(dtype)
    odd = flat[3:].view(1, 500, 4, 64)
    assert odd.is_contiguous() and odd.data_ptr() % 16
    out = packed_attention(q, k, v)
    a = torch.autograd.grad(out, (q, k, v), odd, retain_graph=True)
    b = torch.autograd.grad(out, (q, k, v), odd.clone())
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_attention_under_autocast_takes_the_autocast_type():
    from model.mhc_attention import packed_attention
    q = torch.randn(1, 50, 4, 64, device="cuda", requires_grad=True)
    v = torch.randn(1, 50, 4, 64, device="cuda").bfloat16()
    with torch.autocast("cuda", torch.bfloat16):
        out = packed_attention(q, q, v)  # fp32 queries beside bf16 values
    assert out.dtype == torch.bfloat16
    assert torch.equal(out, packed_attention(q.detach().bfloat16(), q.detach().bfloat16(), v))
    g, = torch.autograd.grad(out.float().sum(), q)
    assert g.dtype == torch.float32 and torch.isfinite(g).all()


def test_a_step_counts_as_an_in_place_change():
    """Autograd refuses a backward through a parameter that the step has changed since."""
    from model.mhc_adamw import adamw_step
    p = torch.randn(8, device="cuda", requires_grad=True)
    y = (p * p).sum()
    m, v = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda")
    adamw_step([p], [torch.ones(8, device="cuda")], [m], [v], step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
