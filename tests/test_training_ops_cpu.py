"""Host-side checks of the training-step operators: bad arguments come back as status codes before any CUDA call, and
the Python entry points refuse what the kernels do not take.  Nothing is launched."""

import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from model import _native
    if not os.path.exists(_native.LIB_PATH) or not os.path.exists(_native.HOST_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _native.load_library()


P = ctypes.c_void_p(4096)      # never dereferenced
ODD = ctypes.c_void_p(4097)
SIX = (ctypes.c_int64 * 6)(512, 64, 256, 64, 256, 64)


def attn(lib, dtype=1, T=100, H=8, Hk=4, D=64, strides=SIX, cu=None, batch=0, seqlen=100, scale=0.125, q=P, ws=P,
         ws_bytes=1 << 20):
    return lib.mhc_attn_fwd(q, P, P, dtype, T, H, Hk, D, strides, cu, batch, seqlen, scale, P, None, P, ws, ws_bytes,
                            None)


def test_attention_refusals(lib):
    assert attn(lib, T=0) == 0                    # nothing to do
    assert attn(lib, dtype=7) == -2
    assert attn(lib, H=8, Hk=3) == -3 and b"cannot share" in lib.mhc_last_error()
    assert attn(lib, D=129) == -3 and attn(lib, D=0) == -3
    assert attn(lib, T=-1) == -3 and attn(lib, T=1 << 31) == -3
    assert attn(lib, seqlen=33) == -3             # 100 tokens are not sequences of 33
    for s in (0.0, -1.0, float("inf"), float("nan")):
        assert attn(lib, scale=s) == -3
    assert attn(lib, cu=P, batch=0) == -3
    assert attn(lib, cu=ODD, batch=2) == -4
    assert attn(lib, q=None) == -1 and attn(lib, strides=None) == -1
    assert attn(lib, strides=(ctypes.c_int64 * 6)(512, 64, -1, 64, 256, 64)) == -3
    assert attn(lib, q=ODD) == -4
    assert attn(lib, ws=None) == -5 and attn(lib, ws_bytes=8) == -5
    st = lib.mhc_attn_bwd(P, P, P, P, None, P, P, 1, 100, 8, 4, 64, SIX, None, 0, 100, 0.125, P, P, P, P, 16, None)
    assert st == -5
    st = lib.mhc_attn_bwd(P, P, P, P, None, P, P, 1, 100, 8, 4, 64, SIX, None, 0, 100, 0.125, P, None, P, P, 1 << 24,
                          None)
    assert st == -1


def test_attention_gradients_that_may_be_left_out(lib):
    """dq, or dk and dv together; what is left is checked as ever (here it stops at the workspace)."""
    for dq, dk, dv, want in ((P, None, None, -5), (None, P, P, -5), (None, None, None, -1), (P, None, P, -1),
                             (P, P, None, -1), (None, P, None, -1), (None, ODD, P, -4)):
        assert lib.mhc_attn_bwd(P, P, P, P, None, P, P, 1, 100, 8, 4, 64, SIX, None, 0, 100, 0.125, dq, dk, dv, P, 16,
                                None) == want


def test_attention_workspaces(lib):
    assert lib.mhc_attn_lse_pitch(0) == 0 and lib.mhc_attn_lse_pitch(1) == 128 and lib.mhc_attn_lse_pitch(129) == 256
    assert lib.mhc_attn_fwd_workspace(100000) >= 782 * 4
    assert lib.mhc_attn_bwd_workspace(1000, 8, 4, 64) >= 1024 * 8 * 4
    # few keys to go by: parts of dK and dV are kept apart
    assert lib.mhc_attn_bwd_workspace(1000, 8, 1, 64) >= 8 * 2 * 1000 * 64 * 4
    # the offset of a long row passes 32 bits
    assert lib.mhc_attn_bwd_workspace(1 << 30, 16, 16, 64) >= (1 << 30) * 64


def route(lib, dtype=0, T=10, E=8, rs=8, k=2, logits=P, counts=P, ws=None, n=0):
    return lib.mhc_route_fwd(logits, dtype, T, E, rs, k, 0.1, P, P, counts, P, ws, n, None)


def test_router_refusals(lib):
    assert route(lib, dtype=9) == -2
    assert route(lib, E=0) == -3 and route(lib, E=513, rs=513) == -3
    assert route(lib, k=0) == -3 and route(lib, k=9) == -3
    assert route(lib, rs=7) == -3 and route(lib, T=-1) == -3
    assert route(lib, logits=None) == -1 and route(lib, counts=None) == -1
    assert route(lib, logits=ODD) == -4
    assert route(lib, T=100000) == -5             # more than one block: it needs its workspace
    assert lib.mhc_route_fwd_workspace(10, 8) == 0 and lib.mhc_route_fwd_workspace(100000, 8) > 0
    assert lib.mhc_route_bwd(P, 0, 0, 8, 8, 2, 0.1, P, P, P, P, P, P, None) == 0
    assert lib.mhc_route_bwd(P, 0, 5, 8, 8, 2, 0.1, P, P, P, P, P, ctypes.c_void_p(4104), None) == -4


def tensors(**over):
    f = dict(p=4096, g=4096, m=4096, v=4096, ms=4096, vs=4096, n=10, step=1, pdt=0, gdt=0) | over
    return (ctypes.c_uint64 * 9)(f["p"], f["g"], f["m"], f["v"], f["ms"], f["vs"], f["n"] & (1 << 64) - 1,
                                 f["step"] & (1 << 64) - 1, f["pdt"] | f["gdt"] << 32)


def adamw(lib, t, bits=32, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.1, clip=0.0, ws=None, count=1):
    return lib.mhc_adamw_step(t, count, bits, lr, b1, b2, eps, wd, clip, ws, None, None)


def test_adamw_refusals(lib):
    assert adamw(lib, None, count=0) == 0 and adamw(lib, tensors(n=0, p=0)) == 0
    assert adamw(lib, None) == -1 and adamw(lib, tensors(), count=-1) == -3
    assert adamw(lib, tensors(), bits=16) == -7
    for bad in (dict(lr=-1.0), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(wd=-1.0), dict(lr=float("nan"))):
        assert adamw(lib, tensors(), **bad) == -3
    assert adamw(lib, tensors(step=0)) == -3 and adamw(lib, tensors(n=-5)) == -3
    assert adamw(lib, tensors(pdt=5)) == -2 and adamw(lib, tensors(gdt=5)) == -2
    for name in ("p", "g", "m", "v"):
        assert adamw(lib, tensors(**{name: 0})) == -1
        assert adamw(lib, tensors(**{name: 4098})) == -4
    assert adamw(lib, tensors(ms=0), bits=8) == -1
    assert adamw(lib, tensors(), clip=1.0) == -5
    assert lib.mhc_grad_norm(tensors(), 1, 0, P, 8, None) == -5
    assert lib.mhc_adamw_unpack(None, 1, P, P, 10, None) == -1 and lib.mhc_adamw_unpack(P, 1, P, P, -1, None) == -3
    assert lib.mhc_adamw_unpack(None, 1, None, None, 0, None) == 0


def test_adamw_check_answers_as_the_step(lib):
    """The same refusals, without a launch; what the step would take is fine."""
    def ask(t, bits=32, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.1, count=1):
        return lib.mhc_adamw_check(t, count, bits, lr, b1, b2, eps, wd)

    assert ask(tensors()) == 0 and ask(tensors(), bits=8) == 0 and ask(None, count=0) == 0
    for args in (dict(bits=16), dict(count=-1), dict(lr=-1.0), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(wd=-1.0),
                 dict(lr=float("nan"))):
        assert ask(tensors(), **args) == adamw(lib, tensors(), **args) < 0
    for t in (dict(step=0), dict(n=-5), dict(pdt=5), dict(gdt=5), dict(p=0), dict(m=4098)):
        assert ask(tensors(**t)) == adamw(lib, tensors(**t)) < 0


def trained_by_torch(cls=torch.optim.AdamW, dtype=torch.float32, **kind):
    ps = [torch.nn.Parameter(torch.randn(s).to(dtype)) for s in ((5, 3), (300,))]
    opt = cls(ps, lr=1e-3, **kind)
    for _ in range(3):
        for p in ps:
            p.grad = torch.randn_like(p)
        opt.step()
    return ps, opt.state_dict()


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_a_checkpoint_of_torch_is_converted(dtype):
    """Counts become ints, moments fp32; a parameter that was never stepped has no state; options of how torch runs
    its step do not stay behind."""
    from model.mhc_adamw import AdamW
    ps, saved = trained_by_torch(dtype=dtype, betas=(0.8, 0.9), foreach=True)
    del saved["state"][1]
    saved["param_groups"][0]["lr"] = torch.tensor(2e-3)
    opt = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps])
    opt.load_state_dict(saved)
    group, = opt.param_groups
    assert set(group) == {"params", "lr", "betas", "eps", "weight_decay"} and group["betas"] == (0.8, 0.9)
    assert type(group["lr"]) is float and abs(group["lr"] - 2e-3) < 1e-9
    s = opt.state[group["params"][0]]
    assert type(s["step"]) is int and s["step"] == 3 and group["params"][1] not in opt.state
    for name in ("exp_avg", "exp_avg_sq"):
        assert s[name].dtype == torch.float32 and torch.equal(s[name], saved["state"][0][name].float())
        assert s[name].data_ptr() != saved["state"][0][name].data_ptr()


def test_checkpoints_that_cannot_be_continued_are_refused(lib):
    """At the load, and nothing of the optimizer has changed by then."""
    from model.mhc_adamw import AdamW, zero_moment
    ps, saved = trained_by_torch()
    own8 = AdamW(ps, state_bits=8)
    for p in ps:
        own8._state_of(p)
    cases = [(8, saved), (32, own8.state_dict()),
             (32, trained_by_torch(amsgrad=True)[1]), (32, trained_by_torch(maximize=True)[1]),
             (32, trained_by_torch(torch.optim.Adam)[1]), (32, trained_by_torch(torch.optim.Adagrad)[1]),
             (32, trained_by_torch(torch.optim.SGD)[1])]
    _, short = trained_by_torch()
    short["state"][1]["exp_avg"] = torch.zeros(299)
    cases.append((32, short))
    codes = own8.state_dict()
    codes["state"][0] = codes["state"][0] | {"exp_avg": zero_moment(ps[0], False).codes}
    cases.append((8, codes))
    for bits, bad in cases:
        opt = AdamW(ps, lr=0.5, state_bits=bits)
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        assert not opt.state and opt.param_groups[0]["lr"] == 0.5
    opt = AdamW(ps, state_bits=8)
    opt.load_state_dict(own8.state_dict())
    assert opt.state[ps[0]]["exp_avg"].dtype == torch.int8 and opt.state[ps[0]]["step"] == 0


def test_python_refuses_cpu_tensors(lib):
    from model.mhc_adamw import AdamW, adamw_step, unpack_moment
    from model.mhc_attention import packed_attention
    from model.mhc_router import route_topk
    q = torch.randn(4, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        packed_attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        route_topk(torch.randn(3, 4), 2)
    t = torch.zeros(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        adamw_step([t], [t], [t], [t], step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="CUDA"):
        unpack_moment(torch.zeros(3, dtype=torch.int8), torch.zeros(1))
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(t)], state_bits=4)
