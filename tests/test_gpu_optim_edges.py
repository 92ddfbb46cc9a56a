"""Places where the training-step operators (v2e2v_amd/optim.py) lose what the formula keeps, or take what
they should refuse: small decay rates of the moments, a 16-bit value's one rounding, small decoupled decay,
state that outlives its parameter's type, views that share memory, and tensors past the cache's size.

U = 2^-24 is half a step of float32 relative to the value; the helpers and the two ways that each test
takes are those of tests/test_gpu_optim.py.
"""
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_optim import (DEV, HYPER, ODD, SPARE, TYPES, U, adam64, adam_case, check_scaled, check_step, gen,  # noqa: F401
                                  make, near, norm64, params_of, params_of_views, snapshot, some, way)
from v2e2v_amd import _lib, optim

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- moments of small rates
def wide_case(dtype, seed):
    """Gradients over nine orders of magnitude beside moments of about 1."""
    ps = []
    for i, n in enumerate((1, 5, 1023, 4097)):
        p = torch.nn.Parameter((torch.rand(n, device=DEV, generator=gen(seed + i)) + 0.5).to(dtype))
        mag = 10.0 ** (-9.0 * torch.rand(n, device=DEV, generator=gen(seed + 10 + i), dtype=torch.float64))
        p.grad = (mag * torch.randn(n, device=DEV, generator=gen(seed + 20 + i)).sign()).to(dtype)
        ps.append(p)
    state = {i: dict(step=torch.tensor(3.0), exp_avg=torch.randn(p.shape, device=DEV, generator=gen(seed + 30 + i)),
                     exp_avg_sq=torch.rand(p.shape, device=DEV, generator=gen(seed + 40 + i)),
                     **({} if dtype == torch.float32 else {"master": p.detach().float()})) for i, p in enumerate(ps)}
    return ps, state


@pytest.mark.parametrize("b1", [0.0, 1e-9, 0.1, 0.3, 0.49])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_first_moment_of_a_small_beta1(dtype, b1):
    """The old moment counts with b1, its roundings too.  b1 m + (1 - b1) g: b1, its product's sum and 1 - b1 are
    off by U each, the product (1 - b1) g too, and the sum by U of the result:
    U (2 b1 |m| + 3 (1 - b1) |g|), plus half of the smallest number for each of two results."""
    ps, state = wide_case(dtype, 7)
    opt = make(ps, state, dict(HYPER, betas=(b1, 0.999)))
    before = snapshot(opt, ps, state)
    opt.step()
    for p, (w, m, v) in zip(ps, before):
        m, g = m.double(), p.grad.double()
        off = (opt.state[p]["exp_avg"].double() - (b1 * m + (1 - b1) * g)).abs()
        bound = SPARE * U * (2 * b1 * m.abs() + 3 * (1 - b1) * g.abs()) + 2.0 ** -149
        assert bool((off <= bound).all()), float((off / bound).max())


def test_steps_of_both_betas_zero():
    """betas (0, 0): whatever the moments were, the step is lr g / (|g| + eps).  With m = g exactly and v off by
    U, the root by half of that, by U and by U of eps and the sum, and the division by U, the step is off by 4 U,
    and the sum by U of the weight."""
    ps, state = wide_case(torch.float32, 17)
    hyper = dict(HYPER, betas=(0.0, 0.0), lr=0.25, eps=1e-5)
    opt = make(ps, state, hyper)
    before = snapshot(opt, ps, state)
    opt.step()
    for p, (w, m, v) in zip(ps, before):
        g = p.grad.double()
        step = 0.25 * g / (g.abs() + 1e-5)
        want = w.double() - step
        assert torch.equal(opt.state[p]["exp_avg"], p.grad)
        off = (p.detach().double() - want).abs()
        assert bool((off <= SPARE * U * (4 * step.abs() + want.abs())).all())


@pytest.mark.parametrize("b2", [1e-9, 0.001, 0.1, 0.3, 0.49])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_second_moment_of_a_small_beta2(dtype, b2):
    """As for the first: b2, its product with v and the sum are off by U each, and so are 1 - b2, its product with
    g and the sum: 3 U of either term."""
    ps, state = wide_case(dtype, 27)
    opt = make(ps, state, dict(HYPER, betas=(0.9, b2)))
    before = snapshot(opt, ps, state)
    opt.step()
    for p, (w, m, v) in zip(ps, before):
        v, g = v.double(), p.grad.double()
        want = b2 * v + (1 - b2) * g * g
        off = (opt.state[p]["exp_avg_sq"].double() - want).abs()
        bound = SPARE * 3 * U * want + 2.0 ** -149
        assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("b2", [0.0, 0.3, 0.9])
def test_an_overflowed_second_moment_stays_infinite(b2):
    """Its weights stay where they are, and its neighbours go on."""
    p = torch.nn.Parameter(torch.ones(4099, device=DEV))
    opt = optim.Adam([p], lr=0.1, betas=(0.9, b2))
    big = torch.zeros(4099, dtype=torch.bool, device=DEV)
    big[[0, 1027, 4098]] = True
    for scale in (1e21, 1.0):
        p.grad = torch.where(big, scale, 1.0)
        opt.step()
    v = opt.state[p]["exp_avg_sq"]
    assert bool(v[big].isinf().all()) and bool((p.detach()[big] == 1.0).all())
    assert bool(((v[~big] - 1.0).abs() < 1.0).all()) and bool((p.detach()[~big] < 0.9).all())


# ------------------------------------------------------------------------------------- one rounding
def near_ties(dtype, seed):
    """A scale c (float32) and values g of the type for which the float32 product, rounded to the type, differs from
    the exact product rounded at once (for bfloat16, which no instruction rounds at once, any values)."""
    r = np.random.default_rng(seed)
    if dtype == torch.bfloat16:
        return float(np.float32(r.uniform(0.5, 1.0))), torch.randn(4096, device=DEV, generator=gen(seed)).to(dtype)
    g = np.arange(1024, 2048) * 2.0 ** -10                    # every significand of float16
    for c in r.uniform(0.5, 1.0, 4000).astype(np.float32):
        exact = g * float(c)                                  # 11 and 24 bits: exact in float64
        hit = g[exact.astype(np.float16) != exact.astype(np.float32).astype(np.float16)]
        if len(hit) >= 2:
            return float(c), torch.tensor(np.concatenate([hit, -hit, 4 * hit]), device=DEV).to(dtype)
    raise AssertionError("no such scale")


@pytest.mark.parametrize("seed", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_clipped_values_do_not_depend_on_their_place(dtype, seed):
    """A 16-bit gradient is the float32 product rounded once, bit for bit, inside a tensor and at its ends."""
    c, values = near_ties(dtype, seed)
    sizes = [1, 3, 7, 8, 9, 15, 16, 33, 1, 1000, 4097, 8191, 30011]
    total = sum(sizes) + 1
    flat = values[torch.randint(len(values), (total,), device=DEV, generator=gen(seed))]
    grads, at = [], 1
    for n in sizes:
        grads.append(flat[at:at + n])
        at += n
    want = [(g.float() * c).to(dtype) for g in grads]
    norm = torch.tensor(2.0, device=DEV)
    optim.clip_grads_with_norm_(params_of(grads), c * (2.0 + 1e-6), norm)
    for g, w in zip(grads, want):
        assert torch.equal(g, w), (g.numel(), int((g != w).sum()))


# ------------------------------------------------------------------------------------- small decay
@pytest.mark.parametrize("lr,wd", [(1e-4, 0.01), (1e-5, 0.01), (2e-6, 0.01)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_decoupled_decay_over_many_steps(dtype, lr, wd):
    """The mean weight of many after many steps.  Each step rounds a weight of [0.5, 1) by at most 2^-25, to either
    side as the update's low bits fall (a deviation of 2^-24 / sqrt(12) each), so the mean of N weights is off by
    2^-24 sqrt(K / (12 N)) in K steps: 8 of them, and 10 U of the updates' sum of magnitudes, are allowed.
    lr wd rounded to multiples of 2^-24 instead is off by 1 % to 100 % of the decay."""
    N, K = 200_000, 40
    p = torch.nn.Parameter((0.6 + 0.3 * torch.rand(N, device=DEV, generator=gen(1))).to(dtype))
    w = p.detach().double()
    m = torch.randn(N, device=DEV, generator=gen(2)) * 0.3
    v = 0.5 + torch.rand(N, device=DEV, generator=gen(3))
    state = {0: dict(step=torch.tensor(1000.0), exp_avg=m.clone(), exp_avg_sq=v.clone(),
                     **({} if dtype == torch.float32 else {"master": p.detach().float()}))}
    b1, b2 = 0.9, 0.999
    opt = make([p], state, dict(HYPER, lr=lr, weight_decay=wd, decoupled=True))
    m, v, start, moved = m.double(), v.double(), w.mean().item(), 0.0
    for k in range(K):
        g = torch.randn(N, device=DEV, generator=gen(100 + k)).to(dtype)
        p.grad = g
        opt.step()
        g, t = g.double(), 1001 + k
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        step = lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + 1e-8)
        w = w * (1 - lr * wd) - step
        moved += step.abs().mean().item()
    got = opt.state[p]["master"] if dtype != torch.float32 else p.detach()
    assert 0.5 < float(got.min()) and float(got.max()) < 1.0
    off = abs(got.double().mean().item() - w.mean().item())
    allowed = 8 * 2.0 ** -24 * math.sqrt(K / (12 * N)) + 10 * U * moved
    assert allowed < 0.01 * K * lr * wd * start                        # what the bound can tell
    assert off <= allowed, (off, allowed, K * lr * wd * start)


@pytest.mark.parametrize("decay", [0.25, 0.49, 0.5, 0.75, 1.0])
def test_large_decoupled_decay(decay):
    """Where little of the old weight is left, its roundings count with what is left: decay is off by U (of 1 - decay
    or of itself, below 1/2, where 1 - decay is at least as large), its product by U, the sum by U of the result, and
    the update by 8 U."""
    ps, state = wide_case(torch.float32, 37)
    hyper = dict(HYPER, lr=1.0, weight_decay=decay, decoupled=True)
    for s in state.values():
        s["exp_avg"] *= 1e-6
    opt = make(ps, state, hyper)
    before = snapshot(opt, ps, state)
    opt.step()
    for p, (w, m, v) in zip(ps, before):
        m1, v1 = opt.state[p]["exp_avg"].double(), opt.state[p]["exp_avg_sq"].double()
        root = v1.sqrt() / math.sqrt(1 - 0.999 ** 4) + 1e-8
        step = m1 / (1 - 0.9 ** 4) / root
        want = w.double() * (1 - decay) - step
        off = (p.detach().double() - want).abs()
        # lr / (1 - b1^t), the division, the root, its factor and sum, the product and both sums: 8 U of the update
        assert bool((off <= SPARE * U * (8 * step.abs() + 4 * (1 - decay) * w.double().abs()) + 2.0 ** -149).all())


def test_decay_of_infinite_weights():
    """p (1 - lr wd) of an infinity is that infinity; a NaN stays one, and their neighbours are the formula's."""
    hyper = dict(HYPER, lr=1e-2, weight_decay=0.1, decoupled=True)
    ps, state = adam_case([4099], torch.float32, 61, 3)
    bad = torch.tensor([5, 1030, 4098], device=DEV)
    with torch.no_grad():
        ps[0][bad] = torch.tensor([math.inf, -math.inf, math.nan], device=DEV)
    opt = make(ps, state, hyper)
    before = snapshot(opt, ps, state)
    opt.step()
    got = ps[0].detach()[bad].tolist()
    assert got[:2] == [math.inf, -math.inf] and math.isnan(got[2])
    with torch.no_grad():
        for w in (ps[0], before[0][0]):
            w[bad] = 0.0
        w1 = adam64(before[0][0], ps[0].grad, *before[0][1:], 4, 1.0, **hyper)
        off = (ps[0].double() - w1[0]).abs()
        off[bad] = 0.0
        assert bool((off <= w1[3][0]).all())


# ------------------------------------------------------------------------------------- state
def give_grads(ps, k):
    for i, p in enumerate(ps):
        p.grad = torch.randn(p.shape, device=DEV, generator=gen(10 * k + i)).to(p.dtype)


@pytest.mark.parametrize("half", [torch.bfloat16, torch.float16])
def test_a_phase_in_float32_is_not_undone(half):
    """16-bit steps, float32 steps, 16-bit steps: the last ones go on from the float32 weights."""
    net = torch.nn.Sequential(torch.nn.Linear(33, 40), torch.nn.Linear(40, 7)).to(DEV, half)
    ps, hyper = list(net.parameters()), dict(HYPER, lr=0.1)
    opt = make(ps, {}, hyper)
    for t in range(2):
        give_grads(ps, t)
        opt.step()
    net.float()
    for t in range(2, 4):
        give_grads(ps, t)
        before = snapshot(opt, ps, {}) if t > 2 else None
        opt.step()
        assert all("master" not in opt.state[p] for p in ps)
        if before:
            check_step(opt, ps, before, hyper, t + 1, 1.0)
    net.to(half)
    give_grads(ps, 4)
    before = [(p.detach().float(), opt.state[p]["exp_avg"].clone(), opt.state[p]["exp_avg_sq"].clone()) for p in ps]
    opt.step()
    check_step(opt, ps, before, hyper, 5, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_state_loaded_from_a_live_optimizer(dtype):
    """Two optimizers that go on from one state: neither moves the other's moments or step counts."""
    ps, _ = adam_case([5, 3000], dtype, 12, 0)
    a = optim.Adam(ps, lr=0.1)
    a.step()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    b = optim.Adam(qs, lr=0.1)
    b.load_state_dict(a.state_dict())
    kept = {n: [a.state[p][n].clone() for p in ps] for n in a.state[ps[0]]}
    b.step()
    assert all(torch.equal(a.state[p][n], old) for n in kept for p, old in zip(ps, kept[n]))
    a.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and a.state[p]["step"].item() == b.state[q]["step"].item() == 2
        assert all(torch.equal(a.state[p][n], b.state[q][n]) for n in kept)


# ------------------------------------------------------------------------------------- views
def overlapping():
    base = torch.randn(12, 20, device=DEV, generator=gen(9))
    z = torch.complex(base[0], base[1])
    yield "the same strided view twice", base, [base[::2, ::3], base[::2, ::3]]
    yield "a strided and a dense one", base, [base[:, 1:5:2], base[4]]
    yield "a dense and a strided one, far apart in the list", base, [base[4, :3], torch.ones(3, device=DEV), base[3:, 2::7]]
    yield "one element in common", base, [base[:6, :11:5], base[5:, 10::9]]
    yield "a view and its transposed one", base, [base[:5, :5], base[:5, :5].t()]
    yield "a negated view and its base", torch.view_as_real(z), [torch.view_as_real(z)[:, 1], z.conj().imag]
    yield "an overlap with itself beside another", base, [base.reshape(-1).as_strided((4, 4), (2, 3)), base.reshape(-1)[15:16]]


@pytest.mark.parametrize("k", range(7))
def test_strided_gradients_that_share_memory_are_refused(k):
    name, base, grads = list(overlapping())[k]
    kept = base.clone()
    version = [g._version for g in grads]
    for call in (lambda: optim.clip_grad_norm_(params_of_views(grads), 1e-3),
                 lambda: optim.clip_grads_with_norm_(params_of_views(grads), 1e-3, torch.tensor(1.0, device=DEV)),
                 lambda: optim.clip_grad_norm_(params_of_views(grads), 1e-3, error_if_nonfinite=True)):
        with pytest.raises(_lib.CistaError, match="overlap"):
            call()
        assert torch.equal(base, kept), name
    assert [g._version for g in grads] == version
    near(optim.grad_norm(grads), norm64(grads, 2), 2)                    # reading them is allowed


def test_views_that_lie_between_each_other_are_clipped():
    """Columns, halves of rows, real and imaginary parts, every second element: disjoint, in one buffer."""
    base = torch.randn(16, 30, device=DEV, generator=gen(19))
    z = torch.complex(base[0], base[1])
    flat = base.reshape(-1)
    for grads in ([base[:, k] for k in range(30)], [base[:, :7], base[:, 7:]], [z.real, z.imag], [z.real, z.conj().imag],
                  [flat[::2], flat[1::2]], [base[::2, ::2], base[1::2].t(), base[::2, 1::2]], [base[:0, ::2], base[:, ::2]]):
        for limit in (0.5, 0.125):                                       # the first one scales the buffer once only
            old = [g.clone() for g in grads]
            norm = norm64(old, 2)
            near(optim.clip_grad_norm_(params_of_views(grads), limit), norm, 2)
            check_scaled([g.clone() for g in grads], old, min(1.0, limit / (norm + 1e-6)))
            with torch.no_grad():
                base.mul_(8.0)


def negated(t):
    """The same values, as a lazily negated view of their opposites."""
    return t.neg()._neg_view()


def test_negated_views_count_with_their_sign():
    """As the given norm, the learning rate, and the optimizer's state."""
    grads = some([5, 4097], torch.float32, 3)
    old = [g.clone() for g in grads]
    total = negated(torch.tensor(4.0, device=DEV))
    assert total.is_neg() and total.item() == 4.0
    optim.clip_grads_with_norm_(params_of(grads), 1.0, total)
    check_scaled(grads, old, 1.0 / (4.0 + 1e-6))
    for dtype in (torch.float32, torch.bfloat16):
        hyper = dict(HYPER, lr=0.25)
        ps, state = adam_case([5, 3000], dtype, 81, 3)
        opt = make(ps, state, hyper)
        opt.param_groups[0]["lr"] = negated(torch.tensor(0.25, device=DEV))
        for p in ps:
            opt.state[p].update({n: negated(t.to(DEV)) for n, t in opt.state[p].items()})
        before = snapshot(opt, ps, {})
        opt.step()
        check_step(opt, ps, before, hyper, 4, 1.0)


def test_scalars_of_other_sizes_are_refused():
    p = torch.nn.Parameter(torch.ones(3, device=DEV))
    p.grad = torch.ones(3, device=DEV)
    opt = optim.Adam([p])
    for n in (0, 2):
        opt.state[p]["step"] = torch.zeros(n, device=DEV)
        with pytest.raises(_lib.CistaError, match="state step"):
            opt.step()
    del opt.state[p]["step"]
    for n in (0, 2):
        opt.param_groups[0]["lr"] = torch.ones(n, device=DEV)
        with pytest.raises(_lib.CistaError, match="lr as a tensor"):
            opt.step()
    assert torch.equal(p.detach(), torch.ones(3, device=DEV))


def test_a_norm_that_is_a_gradient_is_refused():
    grads = some([5, 4097], torch.float32, 3)
    old = [g.clone() for g in grads]
    with pytest.raises(_lib.CistaError, match="overlaps"):
        optim.clip_grads_with_norm_(params_of(grads), 1e-3, grads[1][7])
    assert all(torch.equal(a, b) for a, b in zip(grads, old))


# --------------------------------------------------------------------------- past the cache's size
GUARD = 3


def flat_of(sizes, dtype, seed, scale, off, draw=torch.randn):
    """Views end to end in one buffer that begins `off` elements in, and the buffer."""
    flat = draw(sum(sizes) + off + GUARD, device=DEV, generator=gen(seed)).mul_(scale).to(dtype)
    got, at = [], off
    for n in sizes:
        got.append(flat[at:at + n])
        at += n
    return got, flat


def large_sizes(count):
    """10.9 M elements in `count` tensors: a few large ones, odd ones, small ones and empty ones."""
    sizes = [n % 97 for n in range(count - 5)] + [1025, 777_777, 1_500_001, 3_600_003]
    return sizes + [10_900_000 - sum(sizes)]


@pytest.mark.parametrize("order", [1, 2, math.inf])
@pytest.mark.parametrize("count", [37, 64, 150])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_steps_with_clipping(dtype, count, order):
    """More bytes than the last-level cache holds: one table and several, one group and two, every array of
    tensors end to end at an odd place of its own, and nothing written beside them."""
    sizes = large_sizes(count)
    assert sum(sizes) * 28 > 256 << 20
    half = dtype != torch.float32
    w, wf = flat_of(sizes, dtype, 1, 0.1, 3)
    g, gf = flat_of(sizes, dtype, 2, 0.3, 1)
    m, mf = flat_of(sizes, torch.float32, 3, 0.1, 5)
    v, vf = flat_of(sizes, torch.float32, 4, 0.05, 2, torch.rand)
    master, af = flat_of(sizes, torch.float32, 5, 0.1, 7) if half else (w, wf)
    ps = [torch.nn.Parameter(x) for x in w]
    for p, x in zip(ps, g):
        p.grad = x
    hyper = dict(HYPER, weight_decay=0.05, decoupled=True)
    kw = dict(lr=hyper["lr"], weight_decay=0.05, max_norm=0.2, norm_type=order)
    opt = optim.AdamW(ps if count != 150 else [dict(params=ps[:80]), dict(params=ps[80:])], **kw)
    steps = torch.full((len(ps),), 6.0, device=DEV)
    for i, p in enumerate(ps):
        opt.state[p] = dict(step=steps[i], exp_avg=m[i], exp_avg_sq=v[i], **({"master": master[i]} if half else {}))
    norm = norm64(g, order)
    before = snapshot(opt, ps, {})
    kept = gf.clone()
    arrays = [wf, mf, vf] + ([af] if half else [])
    ends = [(x[:o].clone(), x[-GUARD:].clone()) for x, o in zip(arrays, (3, 5, 2, 7))]
    opt.step()
    near(opt.grad_norm, norm, order)
    check_step(opt, ps, before, hyper, 7, min(1.0, 0.2 / (norm + 1e-6)))
    assert torch.equal(gf, kept)
    for x, o, (a, b) in zip(arrays, (3, 5, 2, 7), ends):
        assert torch.equal(x[:o], a) and torch.equal(x[-GUARD:], b)


@pytest.mark.parametrize("order", [1, 2, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_norms_of_more_than_the_cache_holds(dtype, order):
    size = 2 if dtype != torch.float32 else 4
    n = (280 << 20) // size
    ts, _ = flat_of([5, n // 3, 1, n // 2, 999, n // 6], dtype, 8, 1e-3 if order == 1 else 1.0, 1)
    assert sum(t.numel() for t in ts) * size > 256 << 20
    near(optim.grad_norm(ts, order), norm64(ts, order), order)
