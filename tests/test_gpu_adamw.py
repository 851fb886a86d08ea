"""AdamW step against its formula in 64 bits, the 8-bit moments against a plain fp32 form of their packing.

Tolerances: the fp32 step is about 14 rounded operations a value; m, v and the update are sums of two products, so an
error is at most 16 * 2^-24 of the largest term, plus the parameter's own rounding (half an ulp).  An 8-bit moment
equals the plain fp32 form's code for code: both do the same single IEEE operations."""

import copy
import math
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from model.mhc_adamw import AdamW, adamw_step, adamw_step_8bit, unpack_moment, zero_moment

HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
QB = 256


def make(sizes, dtype, gdtype=None, seed=0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(n, dt, scale, square=False):
        x = torch.randn(n + offset, device="cuda", generator=g) * scale
        return (x.square() if square else x).to(dt)[offset:]

    ps = [t(n, dtype, 0.5) for n in sizes]
    gs = [t(n, gdtype or dtype, 1e-2) for n in sizes]
    ms = [t(n, torch.float32, 3e-3) for n in sizes]
    vs = [t(n, torch.float32, 1e-2, True) for n in sizes]
    return ps, gs, ms, vs


def exact(p, g, m, v, step, lr, betas, eps, weight_decay, factor=1.0):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * factor
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    up = lr / (1 - betas[0] ** step) * m / ((v / (1 - betas[1] ** step)).sqrt() + eps)
    return p * (1 - lr * weight_decay) - up, m, v, up


def compare(old, got, step, dtype, factor=1.0):
    for (p, g, m, v), (p1, m1, v1) in zip(old, got):
        ep, em, ev, up = exact(p, g, m, v, step, factor=factor, **HYPER)
        e = 16 * 2.0 ** -24
        assert ((m1.double() - em).abs() <= e * (m.double().abs() + g.double().abs())).all()
        assert ((v1.double() - ev).abs() <= e * ev + 1e-38).all()
        # the root of v and the quotient carry the relative error of m and v on
        bound = HALF_ULP[dtype] * ep.abs() + e * (p.double().abs() + 16 * up.abs()) + 1e-7 * (dtype == torch.float16)
        assert ((p1.double() - ep).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gdtype", (None, torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("step", (1, 2, 1000))
def test_step(dtype, gdtype, step):
    sizes = [1, 3, 255, 256, 257, 4096, 4097, 10000, 0, 24]
    ps, gs, ms, vs = make(sizes, dtype, gdtype, step)
    old = [tuple(x.clone() for x in q) for q in zip(ps, gs, ms, vs)]
    assert adamw_step(ps, gs, ms, vs, step=step, **HYPER) is None
    compare(old, list(zip(ps, ms, vs)), step, dtype)
    assert all(torch.equal(a, b[1]) for a, b in zip(gs, old))


@pytest.mark.parametrize("count", (1, 24, 25, 440, 441, 900))
def test_many_tensors(count):
    sizes = [(7 * i) % 613 + 1 for i in range(count)]
    ps, gs, ms, vs = make(sizes, torch.float32)
    old = [tuple(x.clone() for x in q) for q in zip(ps, gs, ms, vs)]
    norm = adamw_step(ps, gs, ms, vs, step=5, max_grad_norm=0.5, **HYPER)
    want = math.sqrt(sum(g.double().square().sum().item() for g in gs))
    assert abs(norm.item() - want) <= 1e-6 * want
    compare(old, list(zip(ps, ms, vs)), 5, torch.float32, min(1.0, 0.5 / (want + 1e-6)))


@pytest.mark.parametrize("offset", (1, 2, 3, 4, 5))
@pytest.mark.parametrize("dtype", DTYPES)
def test_misaligned_tensors(dtype, offset):
    ps, gs, ms, vs = make([5000, 300], dtype, None, 1, offset)
    old = [tuple(x.clone() for x in q) for q in zip(ps, gs, ms, vs)]
    adamw_step(ps, gs, ms, vs, step=7, **HYPER)
    compare(old, list(zip(ps, ms, vs)), 7, dtype)


def test_only_its_own_values_change():
    big = torch.full((4, 3000), 7.0, device="cuda")
    ps, ms, vs = [big[0, 100:1101]], [big[1, 100:1101]], [big[2, 100:1101]]
    before = big.clone()
    adamw_step(ps, [torch.ones(1001, device="cuda")], ms, vs, step=1, **HYPER)
    big[:3, 100:1101] = before[:3, 100:1101]
    assert torch.equal(big, before)


def test_mixed_types_in_one_call():
    a, b, c = (make([1000, 77], dt, None, i) for i, dt in enumerate(DTYPES))
    lists = [sum((x[i] for x in (a, b, c)), []) for i in range(4)]
    old = [tuple(x.clone() for x in q) for q in zip(*lists)]
    adamw_step(*lists, step=3, **HYPER)
    for i, dt in enumerate(DTYPES):
        compare(old[2 * i:2 * i + 2], list(zip(lists[0], lists[2], lists[3]))[2 * i:2 * i + 2], 3, dt)


def test_a_step_count_for_every_tensor():
    ps, gs, ms, vs = make([300, 300, 300], torch.float32)
    old = [tuple(x.clone() for x in q) for q in zip(ps, gs, ms, vs)]
    adamw_step(ps, gs, ms, vs, step=[1, 2, 50], **HYPER)
    for i, step in enumerate((1, 2, 50)):
        compare([old[i]], [(ps[i], ms[i], vs[i])], step, torch.float32)


@pytest.mark.parametrize("value", (float("nan"), float("inf")))
def test_non_finite_gradients(value):
    """Without clipping they stay in their value; with it the norm, and so everything, is not finite."""
    ps, gs, ms, vs = make([600, 600], torch.float32)
    gs[0][17] = value
    adamw_step(ps, gs, ms, vs, step=1, **HYPER)
    bad = ~torch.isfinite(ps[0])
    assert bad.sum() == 1 and bad[17] and torch.isfinite(ps[1]).all()
    ps, gs, ms, vs = make([600, 600], torch.float32)
    gs[0][17] = value
    norm = adamw_step(ps, gs, ms, vs, step=1, max_grad_norm=1.0, **HYPER)
    assert not math.isfinite(norm.item()) and torch.isnan(ms[0][17])


def test_clipping_leaves_small_gradients_alone():
    a, b = make([5000], torch.float32, seed=1), make([5000], torch.float32, seed=1)
    adamw_step(*a, step=1, **HYPER)
    norm = adamw_step(*b, step=1, max_grad_norm=1e6, **HYPER)
    assert torch.equal(a[0][0], b[0][0]) and norm.item() < 1e6


# ---- 8 bits --------------------------------------------------------------------

def blocks(x):
    n = x.numel()
    return torch.nn.functional.pad(x.flatten(), (0, -n % QB)).view(-1, QB)


def pack_plain(x, signed):
    b = blocks(x)
    scale = b.abs().amax(1)
    part = b.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    if signed:
        c = (part.sqrt() * 127.0).round() * b.sign()
    else:
        c = (part.sqrt().sqrt() * 255.0).round()
        c = torch.where(b > 0, c.clamp(min=1), c)
    return c.flatten()[:x.numel()].to(torch.int8 if signed else torch.uint8), scale


def unpack_plain(codes, scale, signed):
    c = blocks(codes.float())
    v = c * c.abs() * scale[:, None] * (1 / 16129) if signed else \
        c * c * scale[:, None] * (1 / 65025) * (c * c) * (1 / 65025)
    return v.flatten()[:codes.numel()]


def step_plain(p, g, m, v, step, lr, betas, eps, weight_decay):
    g = g.float()
    m = m * betas[0] + g * (1 - betas[0])
    v = v * betas[1] + g * (1 - betas[1]) * g
    den = v.sqrt() * (1 / math.sqrt(1 - betas[1] ** step)) + eps
    return p.float() * (1 - lr * weight_decay) - m / den * (lr / (1 - betas[0] ** step)), m, v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", (0, 1))
def test_8bit_steps_equal_the_plain_form(dtype, offset):
    sizes = [1, 100, 256, 257, 5000, 4096 * 3 + 5]
    ps, _, _, _ = make(sizes, dtype, offset=offset)
    ms, vs = [zero_moment(p, True) for p in ps], [zero_moment(p, False) for p in ps]
    mine = [(p.clone(), *zero_moment(p, True), *zero_moment(p, False)) for p in ps]
    for step in range(1, 6):
        _, gs, _, _ = make(sizes, dtype, seed=step, offset=offset)
        adamw_step_8bit(ps, gs, ms, vs, step=step, **HYPER)
        for i, (p, mc, msc, vc, vsc) in enumerate(mine):
            p2, m, v = step_plain(p, gs[i], unpack_plain(mc, msc, True), unpack_plain(vc, vsc, False), step, **HYPER)
            mine[i] = (p2.to(dtype), *pack_plain(m, True), *pack_plain(v, False))
            got = (ps[i], ms[i][0], ms[i][1], vs[i][0], vs[i][1])
            assert all(torch.equal(a, b) for a, b in zip(got, mine[i])), (step, i)
    for p, (c, s), (d, r) in zip(ps, ms, vs):
        assert torch.equal(unpack_moment(c, s), unpack_plain(c, s, True))
        assert torch.equal(unpack_moment(d, r), unpack_plain(d, r, False))


def test_8bit_moments_are_near_the_32bit_ones():
    """Spacing of the codes: m is off by at most half a step of the root, (sqrt(|m|/s) / 127 + 1 / 254^2) s, v by
    4 (v/s)^(3/4) / 510 s to first order; both hold with 10 % for the higher orders."""
    ps, gs, _, _ = make([QB * 40], torch.float32)
    ms, vs = [zero_moment(ps[0], True)], [zero_moment(ps[0], False)]
    adamw_step_8bit(ps, gs, ms, vs, step=1, **HYPER)
    m, v = gs[0] * 0.1, gs[0].square() * 0.05
    for got, want, signed in ((unpack_moment(*ms[0]), m, True), (unpack_moment(*vs[0]), v, False)):
        s = blocks(want).abs().amax(1, keepdim=True)
        part = blocks(want).abs() / s
        off = (blocks(got) - blocks(want)).abs() / s
        bound = part.sqrt() / 127 + 1 / 254 ** 2 if signed else 4 * part ** 0.75 / 510 + 1 / 255 ** 2
        assert (off <= 1.1 * bound + 1e-6).all()
    assert (unpack_moment(*vs[0])[v > 0] > 0).all()


def test_8bit_zeros_and_non_finite():
    p = torch.zeros(1000, device="cuda")
    ms, vs = [zero_moment(p, True)], [zero_moment(p, False)]
    adamw_step_8bit([p], [torch.zeros(1000, device="cuda")], ms, vs, step=1, **HYPER)
    assert (p == 0).all() and (ms[0][0] == 0).all() and (vs[0][0] == 0).all()
    for bad in (float("nan"), float("inf")):
        p = torch.zeros(1000, device="cuda")
        ms, vs = [zero_moment(p, True)], [zero_moment(p, False)]
        g = torch.ones(1000, device="cuda")
        g[300] = bad
        adamw_step_8bit([p], [g], ms, vs, step=1, **HYPER)
        m = unpack_moment(*ms[0])
        assert torch.isnan(m[256:512]).all() and torch.isfinite(m[:256]).all() and torch.isfinite(m[512:]).all()


# ---- the optimizer -------------------------------------------------------------

def test_optimizer_follows_torch():
    """fp32, ten steps beside torch.optim.AdamW with clip_grad_norm_, two groups, one parameter without a gradient in
    some steps.  Both are fp32 evaluations of one formula: after ten steps of at most lr each, within 1e-5 of lr-sized
    moves plus 16 roundings of the parameter a step."""
    torch.manual_seed(0)
    mine = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((64, 33), (5,), (300, 7), (1,))]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    groups = lambda ps: [dict(params=ps[:2], weight_decay=0.0), dict(params=ps[2:], lr=1e-2)]  # noqa: E731
    a = AdamW(groups(mine), lr=1e-3, weight_decay=0.1, max_grad_norm=1.0)
    b = torch.optim.AdamW(groups(theirs), lr=1e-3, weight_decay=0.1)
    for step in range(10):
        for i, (p, q) in enumerate(zip(mine, theirs)):
            g = None if i == 1 and step in (2, 3) else torch.randn_like(p)
            p.grad, q.grad = g, None if g is None else g.clone()
        norm = torch.nn.utils.clip_grad_norm_(theirs, 1.0)
        a.step()
        b.step()
        assert abs(a.grad_norm.item() - norm.item()) <= 1e-5 * norm.item()
    for p, q in zip(mine, theirs):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_optimizer_state_survives_saving(bits, dtype):
    torch.manual_seed(1)
    p = torch.nn.Parameter(torch.randn(700, device="cuda").to(dtype))
    opt = AdamW([p], state_bits=bits)
    for _ in range(3):
        p.grad = torch.randn_like(p)
        opt.step()
    p2 = torch.nn.Parameter(p.detach().clone())
    opt2 = AdamW([p2], state_bits=bits)
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))
    for _ in range(2):
        g = torch.randn_like(p)
        p.grad, p2.grad = g.clone(), g.clone()
        opt.step()
        opt2.step()
    assert torch.equal(p, p2)
    for k, v in opt.state[p].items():
        w = opt2.state[p2][k]
        assert v.dtype == w.dtype and torch.equal(v, w) if torch.is_tensor(v) else v == w


@pytest.mark.parametrize("bits", (32, 8))
def test_a_copied_optimizer_steps_as_the_first(bits):
    p = torch.nn.Parameter(torch.randn(600, device="cuda"))
    opt = AdamW([p], state_bits=bits, max_grad_norm=0.1)
    p.grad = torch.randn_like(p)
    opt.step()
    for clone in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        q = clone.param_groups[0]["params"][0]
        assert (clone.state_bits, clone.max_grad_norm) == (bits, 0.1) and torch.equal(clone.grad_norm, opt.grad_norm)
        old = q.detach().clone()
        q.grad = p.grad.clone()
        clone.step()
        assert not torch.equal(q, old) and clone.state[q]["step"] == 2
    opt.step()
    assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("kind", ({}, dict(fused=True), dict(capturable=True)))
def test_goes_on_from_a_checkpoint_of_torch(dtype, kind):
    """Five steps of torch's optimizer, then five of each from its checkpoint.  fp32: as above.  bf16: torch rounds its
    moments and every operation to bf16: 16 roundings of 2^-9 of an update (at most 1.5 lr
    here) and three roundings of the parameter a step, its decay apart."""
    torch.manual_seed(2)
    theirs = [torch.nn.Parameter(torch.randn(s, device="cuda").to(dtype)) for s in ((40, 33), (7,))]
    b = torch.optim.AdamW(theirs, lr=1e-3, weight_decay=0.1, **kind)
    for _ in range(5):
        for p in theirs:
            p.grad = torch.randn_like(p)
        b.step()
    mine = [torch.nn.Parameter(p.detach().clone()) for p in theirs]
    a = AdamW(mine, lr=5.0)
    a.load_state_dict(copy.deepcopy(b.state_dict()))
    assert all(s["step"] == 5 and type(s["step"]) is int and s["exp_avg"].dtype == torch.float32
               for s in a.state.values())
    for _ in range(5):
        for p, q in zip(mine, theirs):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        a.step()
        b.step()
    for p, q in zip(mine, theirs):
        if dtype == torch.float32:
            assert torch.allclose(p, q, rtol=1e-5, atol=1e-6)
        else:
            off = (p.double() - q.double()).abs()
            assert (off <= 5 * (8 * 2.0 ** -8 * 1.5e-3 + 3 * 2.0 ** -8 * q.double().abs())).all()


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("bad", (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0)))
def test_a_refused_step_changes_nothing(bits, bad):
    """The second group's options are out of range: no parameter, moment or count of the first has moved either, and
    the step that follows is the one that a fresh optimizer makes."""
    def build():
        torch.manual_seed(5)
        ps = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in (700, 33)]
        for p in ps:
            p.grad = torch.randn_like(p)
        return ps, AdamW([dict(params=[p]) for p in ps], state_bits=bits, max_grad_norm=1.0, **HYPER)

    (ps, opt), (qs, ref) = build(), build()
    opt.step()
    ref.step()
    flat = lambda o, params: [x.clone() if torch.is_tensor(x) else x for p in params  # noqa: E731
                              for x in (p.detach(), *o.state[p].values())]
    before, versions = flat(opt, ps), [p._version for p in ps]
    good = {k: opt.param_groups[1][k] for k in bad}
    opt.param_groups[1].update(bad)
    with pytest.raises(RuntimeError):
        opt.step()
    same = lambda a, b: all(torch.equal(x, y) if torch.is_tensor(x) else x == y for x, y in zip(a, b))  # noqa: E731
    assert same(before, flat(opt, ps)) and versions == [p._version for p in ps]
    opt.param_groups[1].update(good)
    opt.step()
    ref.step()
    assert same(flat(opt, ps), flat(ref, qs))


def test_on_another_stream():
    a, b = make([100000], torch.float32, seed=2), make([100000], torch.float32, seed=2)
    adamw_step(*a, step=1, max_grad_norm=0.1, **HYPER)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        adamw_step(*b, step=1, max_grad_norm=0.1, **HYPER)
    s.synchronize()
    assert all(torch.equal(x, y) for i in (0, 2, 3) for x, y in zip(a[i], b[i]))


def test_refusals():
    ps, gs, ms, vs = make([10], torch.float32)
    ok = dict(step=1, **HYPER)
    assert adamw_step([], [], [], [], **ok) is None
    with pytest.raises(ValueError):
        adamw_step(ps, [], ms, vs, **ok)
    with pytest.raises(ValueError):
        adamw_step(ps, [gs[0][:9]], ms, vs, **ok)
    with pytest.raises(ValueError):
        adamw_step([torch.zeros(4, 4, device="cuda").t()[1:]], [torch.zeros(12, device="cuda")], [ms[0]], [vs[0]], **ok)
    with pytest.raises(TypeError):
        adamw_step([ps[0].double()], gs, ms, vs, **ok)
    with pytest.raises(TypeError):
        adamw_step(ps, gs, [ms[0].bfloat16()], vs, **ok)
    with pytest.raises((RuntimeError, ValueError)):
        adamw_step([ps[0].cpu()], gs, ms, vs, **ok)
    with pytest.raises(ValueError):
        adamw_step(ps, [gs[0].cpu()], ms, vs, **ok)
    with pytest.raises(ValueError):
        adamw_step(ps, gs, ms, vs, step=1, max_grad_norm=0.0, **HYPER)
    for bad in (dict(step=0), dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(weight_decay=-0.1)):
        with pytest.raises(RuntimeError):
            adamw_step(ps, gs, ms, vs, **{**ok, **bad})
    with pytest.raises(ValueError):
        adamw_step_8bit(ps, gs, [(torch.zeros(10, dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda"))],
                        [zero_moment(ps[0], False)], **ok)
    with pytest.raises(TypeError):
        adamw_step_8bit(ps, gs, [zero_moment(ps[0], False)], [zero_moment(ps[0], False)], **ok)
    with pytest.raises(ValueError):
        unpack_moment(torch.zeros(257, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(TypeError):
        unpack_moment(torch.zeros(10, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(ps[0])], state_bits=16)
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(ps[0])], max_grad_norm=-1)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(g):
            adamw_step(ps, gs, ms, vs, **ok)
