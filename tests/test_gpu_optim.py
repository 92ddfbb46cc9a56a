"""Gradient norm, clipping and the Adam step (v2e2v_amd/optim.py) against their formulas in float64.

Tolerances count roundings, u = 2^-24 being half a step of float32 relative to the value:

* norm: float64 sums, one rounding to float32: u (the sums' own error, under n 2^-53, is covered by
  the 1 % on top); the largest magnitude is exact;
* clipping: the scale comes from the rounded norm (u) and is rounded (u), the product is (u): 3 u,
  plus eps / 2 of a 16-bit type, plus half of the type's smallest number where results get that small;
* Adam: see adam_bounds.
"""
import math
import random

import pytest
import torch

from v2e2v_amd import _lib, optim

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SPARE = 1.01
TYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
DEV = "cuda"

# numbers of elements: around a thread's 4 and 8, a wave, a 1024-element and a 16 KB chunk; empty ones
ODD = [1, 2, 3, 5, 7, 8, 9, 0, 63, 65, 255, 257, 1023, 1024, 1025, 4095, 4096, 4097, 8191, 8192, 8193, 0, 30011]


@pytest.fixture(autouse=True, params=["short", "python"])
def way(request, monkeypatch):
    """Each test through csrc/cista_torch.cpp where it takes the call, and through Python alone."""
    if request.param == "python":
        monkeypatch.setattr(optim, "_short", lambda *args: NotImplemented)
    return request.param


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def some(sizes, dtype, seed, scale=1.0, packed=True):
    """Tensors of these sizes, end to end in one buffer (so at odd places), one element in."""
    flat = torch.randn(sum(sizes) + 1, device=DEV, generator=gen(seed)).mul_(scale).to(dtype)
    if not packed:
        return [torch.randn(n, device=DEV, generator=gen(seed + i)).mul_(scale).to(dtype) for i, n in enumerate(sizes)]
    got, at = [], 1
    for n in sizes:
        got.append(flat[at:at + n])
        at += n
    return got


def norm64(tensors, order):
    flat = torch.cat([t.reshape(-1).double() for t in tensors])
    if not flat.numel():
        return 0.0
    return (flat.square().sum().sqrt() if order == 2 else flat.abs().sum() if order == 1 else flat.abs().max()).item()


def near(norm, want, order):
    assert norm.dtype == torch.float32 and norm.shape == ()
    if order == math.inf:
        assert norm.item() == want
    else:
        # below 2^-126 float32's steps are 2^-149 whatever the value, so half a step is 2^-150
        assert abs(norm.item() - want) <= SPARE * U * want + 2.0 ** -150, (norm.item(), want)


def params_of(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        out.append(p)
    return out


def check_scaled(got, old, c):
    """got = c old with the roundings that the module's text counts."""
    for a, b in zip(got, old):
        want = b.double() * c
        eps = 3 * U + (torch.finfo(a.dtype).eps / 2 if a.dtype != torch.float32 else 0.0)
        off = (a.double() - want).abs()
        assert bool((off <= SPARE * eps * want.abs() + TINY[a.dtype] / 2).all()), float((off / want.abs()).max())


# ------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("order", [1, 2, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_odd_sizes(dtype, order):
    ts = some(ODD, dtype, 1)
    near(optim.grad_norm(ts, order), norm64(ts, order), order)
    for n in ODD:
        t = some([n], dtype, n + 2)
        near(optim.grad_norm(t, order), norm64(t, order), order)
        near(optim.grad_norm(t[0], order), norm64(t, order), order)


@pytest.mark.parametrize("order", [1, 2, math.inf])
@pytest.mark.parametrize("count", [1, 63, 64, 65, 191, 192, 193, 450])
def test_norm_of_many_tensors_of_mixed_types(count, order):
    r = random.Random(count)
    ts = [t for k in range(count) for t in some([r.choice([0, 1, 3, 100, 5000])], TYPES[k % 3], k, 10.0 ** r.randint(-3, 3))]
    near(optim.grad_norm(ts, order), norm64(ts, order), order)


def test_norm_of_strided_tensors():
    base = torch.randn(6, 8, 5, 7, device=DEV, generator=gen(5))
    ts = [base.to(memory_format=torch.channels_last), base.permute(3, 1, 0, 2), base[:, 1:7:2], base[::2, :, 1:4],
          base[0, 0, 0, :1].expand(9, 4), base[2, 3, 1, 2], base]
    near(optim.grad_norm(ts), norm64(ts, 2), 2)
    near(optim.grad_norm([base, base]), norm64([base, base], 2), 2)


def test_norm_of_extreme_values():
    """Squares that float32 does not hold; infinities and NaN, alone and together."""
    for v in (1e25, 1e-30, 2.0 ** -140):
        t = torch.full((1000,), v, device=DEV)
        near(optim.grad_norm(t), norm64([t], 2), 2)
    near(optim.grad_norm(torch.full((9000,), 3e38, device=DEV, dtype=torch.bfloat16)), math.inf, math.inf)
    t = torch.randn(20001, device=DEV)
    for order in (1, 2, math.inf):
        t[12345] = -math.inf
        assert optim.grad_norm([t], order).item() == math.inf
        t[777] = math.nan
        assert math.isnan(optim.grad_norm([t], order).item())
        assert math.isnan(optim.grad_norm([t.bfloat16(), torch.ones(3, device=DEV)], order).item())
        t[12345] = 0.0
        assert math.isnan(optim.grad_norm([t], order).item())
        t[777] = 0.0
    assert optim.grad_norm(torch.zeros(5000, device=DEV)).item() == 0.0
    assert optim.grad_norm([torch.empty(0, device=DEV), torch.empty(0, 3, device=DEV)], math.inf).item() == 0.0


def test_nonfinite_norm_raises_when_asked():
    ps = params_of([torch.tensor([1.0, math.inf], device=DEV)])
    with pytest.raises(RuntimeError, match="not finite"):
        optim.grad_norm([ps[0].grad], error_if_nonfinite=True)
    with pytest.raises(RuntimeError, match="not finite"):
        optim.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert ps[0].grad.tolist() == [1.0, math.inf]
    ps[0].grad[1] = 1.0
    assert abs(optim.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True).item() - math.sqrt(2)) <= SPARE * U * math.sqrt(2)
    assert abs(ps[0].grad[0].item() - 1 / (math.sqrt(2) + 1e-6)) <= SPARE * 3 * U


# ------------------------------------------------------------------------------------- clipping
@pytest.mark.parametrize("order", [1, 2, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_clipping(dtype, order):
    grads = some(ODD, dtype, 11, 0.5)
    old = [g.clone() for g in grads]
    norm = norm64(old, order)
    before = [g._version for g in grads]
    near(optim.clip_grad_norm_(params_of(grads), 10 * norm, order), norm, order)      # within the limit
    assert all(torch.equal(a, b) for a, b in zip(grads, old))
    near(optim.clip_grad_norm_(params_of(grads), 0.3 * norm, order), norm, order)
    check_scaled(grads, old, 0.3 * norm / (norm + 1e-6))
    assert all(g._version > v for g, v in zip(grads, before))
    assert optim.clip_grad_norm_(params_of(grads), 0.0, order).item() > 0
    assert all(not g.any() for g in grads)


def test_clipping_by_a_given_norm():
    grads = some([5, 4097, 0, 70000], torch.float32, 3) + some([33, 9001], torch.float16, 4) + some([8193], torch.bfloat16, 5)
    old = [g.clone() for g in grads]
    ps = params_of(grads) + [torch.nn.Parameter(torch.zeros(3, device=DEV))]          # one without a gradient
    for total in (torch.tensor(4.0, device=DEV), torch.tensor([4.0], device=DEV, dtype=torch.float64)):
        for g, o in zip(grads, old):
            g.copy_(o)
        optim.clip_grads_with_norm_(iter(ps), 1.0, total)
        check_scaled(grads, old, 1.0 / (4.0 + 1e-6))
    with pytest.raises(_lib.CistaError, match="scalar tensor"):
        optim.clip_grads_with_norm_(ps, 1.0, torch.tensor(4.0))
    with pytest.raises(_lib.CistaError, match="scalar tensor"):
        optim.clip_grads_with_norm_(ps, 1.0, 4.0)


def test_clipping_is_the_norm_and_then_the_scale():
    a, b = some(ODD, torch.float32, 7), some(ODD, torch.float32, 7)
    norm = optim.clip_grad_norm_(params_of(a), 1.0)
    again = optim.grad_norm(b)
    optim.clip_grads_with_norm_(params_of(b), 1.0, again)
    assert torch.equal(norm, again) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_neighbours_stay_as_they_were():
    """Nothing is written before, between or behind the gradients."""
    for dtype in TYPES:
        buf = torch.randn(100000, device=DEV, generator=gen(8)).to(dtype)
        spans = [(3, 4), (10, 4107), (5001, 5001), (6001, 14195), (20000, 20001), (30001, 77777)]
        old = buf.clone()
        optim.clip_grad_norm_(params_of([buf[a:b] for a, b in spans]), 0.5)
        inside = torch.zeros(100000, dtype=torch.bool, device=DEV)
        for a, b in spans:
            inside[a:b] = True
        assert torch.equal(buf[~inside], old[~inside]) and not torch.equal(buf[inside], old[inside])


def test_clipping_strided_and_shared_gradients():
    base = torch.randn(6, 8, 10, device=DEV, generator=gen(9))
    grads = [base[:, 1:7:2], base[:, ::8, 3:7].transpose(0, 2), base[5, 7, 9]]
    old = [g.clone() for g in grads]
    whole = base.clone()
    norm = norm64(old, 2)
    near(optim.clip_grad_norm_(params_of_views(grads), 1.0), norm, 2)
    check_scaled(grads, old, 1.0 / (norm + 1e-6))
    touched = torch.zeros_like(base, dtype=torch.bool)
    for g in (touched[:, 1:7:2], touched[:, ::8, 3:7], touched[5, 7, 9]):
        g.fill_(True)
    assert torch.equal(base[~touched], whole[~touched])
    t = torch.randn(100, device=DEV)
    for pair in ([t, t], [t[:60], t[59:]], [t[50:], t[:51]]):
        kept = t.clone()
        with pytest.raises(_lib.CistaError, match="overlaps"):
            optim.clip_grad_norm_(params_of(pair), 1e-3)
        assert torch.equal(t, kept)


def params_of_views(grads):
    """Parameters whose gradient is a view of any strides (assigned as such)."""
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, device=DEV))
        p.grad = g
        out.append(p)
    return out


def test_gradients_that_are_odd_views():
    """A gradient that repeats one element is refused before anything is written; a lazily negated one counts
    with its sign."""
    ps = params_of([torch.ones(4, device=DEV)]) + params_of_views([torch.ones(1, device=DEV).expand(6)])
    with pytest.raises(_lib.CistaError, match="overlaps itself"):
        optim.clip_grad_norm_(ps, 1e-3)
    with pytest.raises(_lib.CistaError, match="overlaps itself"):
        optim.clip_grads_with_norm_(ps, 1e-3, torch.tensor(1.0, device=DEV))
    assert torch.equal(ps[0].grad, torch.ones(4, device=DEV))
    near(optim.grad_norm([p.grad for p in ps]), math.sqrt(10.0), 2)
    z = torch.complex(torch.randn(50, device=DEV, generator=gen(2)), torch.randn(50, device=DEV, generator=gen(3)))
    neg = z.conj().imag
    assert neg.is_neg()
    p = params_of_views([neg])[0]
    old, hyper = neg.clone(), dict(HYPER)
    opt = make([p], {}, hyper)
    before = snapshot(opt, [p], {})
    opt.step()
    check_step(opt, [p], before, hyper, 1, 1.0)
    norm = norm64([old], 2)
    near(optim.clip_grad_norm_([p], 0.5), norm, 2)
    check_scaled([p.grad.clone()], [old], 0.5 / (norm + 1e-6))
    flat = torch.view_as_real(z)[:, 1].neg().contiguous()._neg_view()       # dense, and negated
    q = params_of([torch.zeros(50, device=DEV)])[0]
    q.grad = flat
    opt = make([q], {}, hyper)
    before = snapshot(opt, [q], {})
    opt.step()
    check_step(opt, [q], before, hyper, 1, 1.0)


def test_clipping_of_nonfinite_norms():
    g = torch.tensor([1.0, -2.0, math.inf], device=DEV)
    assert optim.clip_grad_norm_(params_of([g]), 1.0).item() == math.inf
    assert g[:2].tolist() == [0.0, 0.0] and math.isnan(g[2].item())
    g = torch.tensor([1.0, -2.0, math.nan], device=DEV, dtype=torch.float16)
    assert math.isnan(optim.clip_grad_norm_(params_of([g]), 1.0).item()) and bool(g.isnan().all())
    g = torch.tensor([1.0, -2.0, math.nan] + [3.0] * 5000, device=DEV, dtype=torch.bfloat16)
    assert math.isnan(optim.clip_grad_norm_(params_of([g]), 1.0).item()) and bool(g.isnan().all())
    g = torch.tensor([1.0, -2.0, math.inf], device=DEV, dtype=torch.bfloat16)
    optim.clip_grad_norm_(params_of([g]), math.inf)                                   # no limit: nothing is scaled
    assert g.tolist() == [1.0, -2.0, math.inf]


# ------------------------------------------------------------------------------------- Adam
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False, maximize=False)


def adam64(w, g, m, v, t, c, lr, betas, eps, weight_decay, decoupled, maximize):
    """One step in float64 from float32 state; t is the step's number. Also the bounds of adam_bounds."""
    b1, b2 = betas
    w, g, m, v = w.double(), g.double() * c, m.double(), v.double()
    if maximize:
        g = -g
    big = g.abs()
    w0 = w
    if decoupled:
        w = w * (1 - lr * weight_decay)
    else:
        big = big + weight_decay * w.abs()
        g = g + weight_decay * w
    m1 = m + (1 - b1) * (g - m)
    v1 = b2 * v + (1 - b2) * g * g
    size, inv = lr / -math.expm1(t * math.log(b1)) if b1 else lr, 1 / math.sqrt(-math.expm1(t * math.log(b2)) if b2 else 1.0)
    root = v1.sqrt() * inv + eps
    w1 = w - size * m1 / root
    return w1, m1, v1, adam_bounds(w0, big, m, v, m1, v1, w1, size, inv, root, 1 - b1, 1 - b2)


def adam_bounds(w0, big, m, v, m1, v1, w1, size, inv, root, r1, r2):
    """Bounds of the float32 step's errors, with G = |c g| + |wd w| (`big`):
    g:  the scale is off by 2 u (its norm, itself), the product by u; wd and the fma by u each: 4 u G
    m': the difference is off by 4 u G + u (G + |m|), 1 - b1 by u, the fma by u |m'|:
        r1 (6 u G + 2 u |m|) + u (|m| + r1 (G + |m|)) <= 8 u (|m| + r1 G)
    v': v - r2 v by u v + u r2 v, r2 g twice u, g 4 u twice, the fma by u: <= 12 u (v + r2 G^2)
    the root: half of v' relative error, sqrt, 1/sqrt(1 - b2^t) and the fma by u each
    w': lr/(1 - b1^t) and the division by u each, the decay's factor and product by u |w| each, the fma by
        u |w'|."""
    em = 8 * U * (m.abs() + r1 * big)
    ev = 12 * U * (v + r2 * big * big) + 2.0 ** -149
    er = torch.where(v1 > 0, ev / (2 * v1.clamp(min=1e-300).sqrt()), torch.zeros_like(v1)) * inv + 3 * U * root
    off = torch.where(root > 0, (em + m1.abs() * er / root) / root, torch.zeros_like(root)) * size
    ew = off + 3 * U * size * (m1 / root).abs() + 2 * U * w0.abs() + U * w1.abs()
    return SPARE * ew + 2.0 ** -149, SPARE * em + 2.0 ** -149, SPARE * ev


def adam_case(sizes, dtype, seed, t):
    ps = params_of(some(sizes, dtype, seed, 0.3))
    state = {}
    for i, p in enumerate(ps):
        with torch.no_grad():
            p.copy_(torch.randn(p.shape, device=DEV, generator=gen(seed + 100 + i)) * 0.1)
        if t:
            state[i] = dict(step=torch.tensor(float(t)), exp_avg=torch.randn(p.shape, device=DEV, generator=gen(seed + 200 + i)) * 0.1,
                            exp_avg_sq=torch.rand(p.shape, device=DEV, generator=gen(seed + 300 + i)) * 0.05)
            if dtype != torch.float32:
                state[i]["master"] = p.detach().float() * (1 + 2.0 ** -12)
    return ps, state


def make(ps, state, hyper, **kw):
    h = dict(hyper)
    decoupled = h.pop("decoupled")
    opt = optim.Adam(ps, decoupled_weight_decay=decoupled, **h, **kw)
    if state:
        sd = opt.state_dict()
        sd["state"] = {i: {k: v.clone() for k, v in s.items()} for i, s in state.items()}
        opt.load_state_dict(sd)
    return opt


def check_step(opt, ps, before, hyper, t, c):
    """The state after one step against the formula from the state before it."""
    for p, (w, m, v) in zip(ps, before):
        st = opt.state[p]
        w1, m1, v1, (ew, em, ev) = adam64(w, p.grad, m, v, t, c, **hyper)
        new = st["master"] if p.dtype != torch.float32 else p.detach()
        assert st["step"].item() == t and st["step"].dtype == torch.float32
        for name, a, b, e in (("m", st["exp_avg"], m1, em), ("v", st["exp_avg_sq"], v1, ev), ("w", new, w1, ew)):
            off = (a.double() - b).abs()
            assert bool((off <= e).all()), (name, float((off / e).max()))
        if p.dtype != torch.float32:
            assert torch.equal(p.detach(), new.to(p.dtype))


def snapshot(opt, ps, state):
    out = []
    for i, p in enumerate(ps):
        s = opt.state.get(p) or state.get(i) or {}
        w = s.get("master", p.detach()).float().clone()
        zero = torch.zeros_like(w)
        out.append((w, s.get("exp_avg", zero).clone(), s.get("exp_avg_sq", zero).clone()))
    return out


@pytest.mark.parametrize("t", [0, 1, 7, 1000])
@pytest.mark.parametrize("hyper", [
    dict(), dict(weight_decay=0.1), dict(weight_decay=0.1, decoupled=True), dict(maximize=True, weight_decay=0.01),
    dict(betas=(0.0, 0.0)), dict(betas=(0.5, 0.9), eps=1e-3, lr=0.0), dict(lr=1.0, weight_decay=0.5, decoupled=True, maximize=True)])
@pytest.mark.parametrize("dtype", TYPES)
def test_adam_step(dtype, hyper, t):
    hyper = dict(HYPER, **hyper)
    ps, state = adam_case(ODD, dtype, 21, t)
    opt = make(ps, state, hyper)
    for k in range(2):
        before = snapshot(opt, ps, state)
        version = [p._version for p in ps]
        kept = [p.grad.clone() for p in ps]
        opt.step()
        check_step(opt, ps, before, hyper, t + k + 1, 1.0)
        assert all(p._version > x for p, x in zip(ps, version))
        assert all(torch.equal(p.grad, g) for p, g in zip(ps, kept)) and opt.grad_norm is None


@pytest.mark.parametrize("order", [1, 2, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_adam_step_with_clipping(dtype, order):
    for limit, active in ((0.2, True), (1e6, False)):
        hyper = dict(HYPER, weight_decay=0.05)
        ps, state = adam_case(ODD, dtype, 31, 5)
        norm = norm64([p.grad for p in ps], order)
        opt = make(ps, state, hyper, max_norm=limit, norm_type=order)
        before = snapshot(opt, ps, state)
        kept = [p.grad.clone() for p in ps]
        opt.step()
        near(opt.grad_norm, norm, order)
        check_step(opt, ps, before, hyper, 6, limit / (norm + 1e-6) if active else 1.0)
        assert all(torch.equal(p.grad, g) for p, g in zip(ps, kept))


@pytest.mark.parametrize("count", [1, 64, 65, 130, 400])
def test_adam_of_many_tensors_in_groups(count):
    """Groups with their own hyperparameters, one norm over all; parameters without a gradient stay."""
    r = random.Random(count)
    sizes = [r.choice([0, 1, 4, 100, 1025, 3000]) for _ in range(count)]
    hypers = [dict(HYPER, lr=1e-2, weight_decay=0.1, decoupled=True), dict(HYPER, lr=1e-3, betas=(0.8, 0.95))]
    ps, _ = adam_case(sizes, torch.float32, 41, 0)
    half = count // 2
    for p in ps[3::7]:
        p.grad = None
    opt = optim.Adam([dict(params=q, lr=h["lr"], betas=h["betas"], weight_decay=h["weight_decay"],
                           decoupled_weight_decay=h["decoupled"]) for q, h in zip((ps[:half], ps[half:]), hypers) if q],
                     max_norm=0.7)
    have = [p for p in ps if p.grad is not None]
    norm = norm64([p.grad for p in have], 2)
    before = snapshot(opt, ps, {})
    opt.step()
    near(opt.grad_norm, norm, 2)
    c = min(1.0, 0.7 / (norm + 1e-6))
    for i, p in enumerate(ps):
        if p.grad is None:
            assert torch.equal(p.detach(), before[i][0]) and p not in opt.state
        else:
            check_step(opt, [p], [before[i]], hypers[0] if i < half else hypers[1], 1, c)


def test_adam_mixed_types_and_layouts():
    """One group of three types; channels-last parameters with gradients in another layout, and the reverse."""
    torch.manual_seed(3)
    ps = []
    for k, dtype in enumerate(TYPES):
        w = torch.randn(6, 4, 3, 5, device=DEV, generator=gen(k)).to(dtype)
        g = torch.randn(6, 4, 3, 5, device=DEV, generator=gen(k + 9)).to(dtype)
        for a, b in ((w.to(memory_format=torch.channels_last), g), (w, g.to(memory_format=torch.channels_last)),
                     (w.permute(3, 0, 2, 1), g.permute(3, 0, 2, 1)), (w, g.new_ones(1).expand_as(g))):
            p = torch.nn.Parameter(a.clone(memory_format=torch.preserve_format))
            p.grad = b.clone(memory_format=torch.preserve_format) if b.stride()[0] else b
            ps.append(p)
    hyper = dict(HYPER, weight_decay=0.1)
    opt = make(ps, {}, hyper, max_norm=3.0)
    norm = norm64([p.grad for p in ps], 2)
    for t in (1, 2):
        before = snapshot(opt, ps, {})
        opt.step()
        check_step(opt, ps, before, hyper, t, 3.0 / (norm + 1e-6))
    with pytest.raises(_lib.CistaError, match="does not fill"):
        p = torch.nn.Parameter(torch.zeros(4, 6, device=DEV)[:, :3])
        p.grad = torch.ones(4, 3, device=DEV)
        optim.Adam([p]).step()


def test_adam_refuses_parameters_that_share_memory():
    base = torch.zeros(50, device=DEV)
    ps = [torch.nn.Parameter(base[:30]), torch.nn.Parameter(base[29:])]
    for p in ps:
        p.grad = torch.ones_like(p)
    with pytest.raises(_lib.CistaError, match="overlaps"):
        optim.Adam(ps).step()
    assert not base.any()
    with pytest.warns(UserWarning, match="duplicate"):
        twice = optim.Adam([ps[0], ps[0]])
    with pytest.raises(_lib.CistaError, match="overlaps"):
        twice.step()
    assert not base.any()


def test_adam_refuses_a_gradient_or_state_of_another_shape():
    """A parameter that was given other data after its gradient, or its state, was made."""
    p = torch.nn.Parameter(torch.ones(6, 4, device=DEV))
    p.grad = torch.ones(6, 4, device=DEV)
    opt = optim.Adam([p])
    opt.step()
    after = p.detach().clone()
    p.data = after[:, :2].contiguous()
    with pytest.raises(_lib.CistaError, match="not like its parameter"):
        opt.step()
    p.grad = torch.ones(6, 2, device=DEV)
    with pytest.raises(_lib.CistaError, match="state exp_avg has shape"):
        opt.step()
    p.data = after.t().contiguous()                       # as many elements, other places
    p.grad = torch.ones(4, 6, device=DEV)
    with pytest.raises(_lib.CistaError, match="state exp_avg has shape"):
        opt.step()
    p.data = after.bfloat16()
    p.grad = torch.ones(6, 4, device=DEV, dtype=torch.bfloat16)
    opt.step()                                            # another type: a master copy is made
    assert opt.state[p]["master"].dtype == torch.float32 and opt.state[p]["step"].item() == 2


def test_adam_of_zero_gradients_and_overflowing_squares():
    p = torch.nn.Parameter(torch.ones(5000, device=DEV))
    p.grad = torch.zeros_like(p)
    opt = optim.Adam([p])
    opt.step()
    assert torch.equal(p.detach(), torch.ones_like(p))
    p.grad.fill_(1e21)                      # its square is not a float32: the average becomes infinite and stays so
    opt.step()
    p.grad.fill_(1.0)
    opt.step()
    assert bool(opt.state[p]["exp_avg_sq"].isinf().all()) and torch.equal(p.detach(), torch.ones_like(p))


def test_folded_clipping_is_clipping_and_then_the_step():
    """For float32 gradients the same numbers, bit for bit, over several steps."""
    runs = []
    for folded in (True, False):
        ps, _ = adam_case(ODD, torch.float32, 51, 0)
        opt = optim.Adam(ps, lr=1e-2, max_norm=0.5 if folded else None)
        for k in range(4):
            for i, p in enumerate(ps):
                p.grad = torch.randn(p.shape, device=DEV, generator=gen(1000 * k + i))
            norm = None if folded else optim.clip_grad_norm_(ps, 0.5)
            opt.step()
            runs.append([p.detach().clone() for p in ps] + [opt.grad_norm if folded else norm])
    for a, b in zip(runs[:4], runs[4:]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_short_way_is_taken(way, monkeypatch):
    """What a training step does goes through csrc/cista_torch.cpp; what that leaves to Python works too."""
    if way == "python":
        pytest.skip("only the short way")
    ps, _ = adam_case([5, 3000], torch.bfloat16, 12, 0)
    opt = optim.Adam([dict(params=ps, lr=torch.tensor(0.1, device=DEV))], max_norm=1.0)
    opt.step()                                            # makes the state, in Python
    taken = []
    real = optim._short
    monkeypatch.setattr(optim, "_short", lambda *a: taken.append(real(*a)) or taken[-1])
    optim.grad_norm([p.grad for p in ps])
    optim.grad_norm(tuple(p.grad for p in ps))
    optim.clip_grad_norm_(iter(ps), 1.0)
    opt.step()
    assert len(taken) == 4 and all(isinstance(t, torch.Tensor) for t in taken)
    ps[0].grad = ps[0].grad.new_ones(10)[::2]
    optim.clip_grad_norm_(ps, 1.0)
    assert taken[-1] is NotImplemented
    ps[0].grad = torch.ones_like(ps[0])
    plain = optim.Adam(ps)
    plain.step()
    plain.step()
    assert taken[-1] is None


def test_equal_inputs_give_equal_bits():
    sizes = [100003, 1, 65, 2000001]
    grads = some(sizes, torch.bfloat16, 6)
    norms = {optim.grad_norm(grads, 2).item() for _ in range(5)} | {optim.grad_norm([g.clone() for g in grads]).item()}
    assert len(norms) == 1


# --------------------------------------------------------------------------- streams, graphs, sizes
def test_side_streams_at_once():
    """Two streams run the operators at the same time, each on its own tensors."""
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [some([300001, 70001, 5], torch.float32, 60 + k) for k in range(2)]
    want = [norm64(s, 2) for s in sets]
    old = [[g.clone() for g in s] for s in sets]
    ps = [params_of(s) for s in sets]
    torch.cuda.synchronize()
    norms = [[], []]
    for k in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                norms[i].append(optim.grad_norm(sets[i]))
                if k == 9:
                    norms[i].append(optim.clip_grad_norm_(ps[i], 1.0))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(abs(n.item() - want[i]) <= SPARE * U * want[i] for n in norms[i])
        check_scaled(sets[i], old[i], 1.0 / (want[i] + 1e-6))


def test_steps_on_a_side_stream():
    """A stream of its own, gradients made on it, and memory freed and reused between the steps."""
    torch.cuda.synchronize()
    runs = []
    for s in (torch.cuda.Stream(), torch.cuda.current_stream()):
        with torch.cuda.stream(s):
            ps, _ = adam_case([70001, 3, 500000], torch.bfloat16, 65, 0)
            opt = optim.AdamW(ps, lr=1e-2, max_norm=0.5)
            for k in range(6):
                for i, p in enumerate(ps):
                    p.grad = torch.randn(p.shape, device=DEV, generator=gen(10 * k + i)).bfloat16()
                opt.step()
                del p
                spill = torch.full((1 << 20,), math.nan, device=DEV)    # what a freed workspace may become
                del spill
            s.synchronize()
            runs.append([p.detach().clone() for p in ps] + [opt.grad_norm])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_captured_steps_replay_like_eager_ones():
    """Two graphs of the same operators, replayed in turn with eager work between, against an eager run."""
    sizes = [1, 3, 4097, 70001, 64]
    shape = lambda: adam_case(sizes, torch.float32, 71, 0)[0]          # noqa: E731
    lr = torch.tensor(1e-2, device=DEV)

    def new_grads(ps, k):
        for i, p in enumerate(ps):
            p.grad.copy_(torch.randn(p.shape, device=DEV, generator=gen(100 * k + i)))

    eager, ps = shape(), shape()
    opts = [optim.Adam(q, lr=lr, max_norm=0.5) for q in (eager, ps)]
    with pytest.raises(_lib.CistaError, match="captured"):             # no state yet
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opts[1].step()
    for q, o in zip((eager, ps), opts):
        new_grads(q, 0)
        o.step()
    torch.cuda.synchronize()
    graphs, norms = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append((optim.clip_grad_norm_(ps, 2.0), optim.grad_norm([p.grad for p in ps], 1)))
            opts[1].step()
            norms[-1] += (opts[1].grad_norm,)
        graphs.append(g)
    for k in range(1, 7):
        lr.fill_(1e-2 / k)
        new_grads(ps, k)
        new_grads(eager, k)
        graphs[k % 2].replay()
        want = (optim.clip_grad_norm_(eager, 2.0), optim.grad_norm([p.grad for p in eager], 1))
        opts[0].step()
        want += (opts[0].grad_norm,)
        if k % 3 == 0:
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(norms[k % 2], want)), k
        for p, q in zip(ps, eager):
            assert torch.equal(p, q) and torch.equal(p.grad, q.grad), k
            assert all(torch.equal(opts[1].state[p][n], opts[0].state[q][n]) for n in ("step", "exp_avg", "exp_avg_sq"))


def test_learning_rate_as_a_tensor():
    ps, state = adam_case([5, 2000], torch.float32, 81, 3)
    qs, _ = adam_case([5, 2000], torch.float32, 81, 3)
    a = make(ps, state, dict(HYPER, lr=torch.tensor(0.5, device=DEV), weight_decay=0.25, decoupled=True))
    b = make(qs, state, dict(HYPER, lr=0.5, weight_decay=0.25, decoupled=True))
    c = make(adam_case([5, 2000], torch.float32, 81, 3)[0], state, dict(HYPER, lr=torch.tensor(0.5), weight_decay=0.25, decoupled=True))
    for o in (a, b, c):
        o.step()
    for p, q, r in zip(ps, qs, c.param_groups[0]["params"]):
        assert torch.equal(p, q) and torch.equal(p, r)
    with pytest.raises(_lib.CistaError, match="float32"):
        make(qs, {}, dict(HYPER, lr=torch.tensor(0.5, device=DEV, dtype=torch.float64))).step()


def test_a_run_taken_up_again():
    """state_dict and load_state_dict in the middle of a run: the same bits as the run that goes on."""
    for dtype in (torch.float32, torch.bfloat16):
        runs = []
        for resume in (False, True):
            ps, _ = adam_case([7, 5000], dtype, 91, 0)
            opt = optim.AdamW(ps, lr=1e-2, max_norm=1.0)
            for k in range(4):
                for i, p in enumerate(ps):
                    p.grad = torch.randn(p.shape, device=DEV, generator=gen(10 * k + i)).to(dtype)
                if resume and k == 2:
                    sd = opt.state_dict()
                    sd["state"] = {i: {n: v.cpu() for n, v in s.items()} for i, s in sd["state"].items()}
                    opt = optim.AdamW(ps, lr=5.0, max_norm=1.0)
                    opt.load_state_dict(sd)
                opt.step()
            runs.append([p.detach().clone() for p in ps])
        assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("kw", [{}, {"foreach": True}, {"fused": True}])
def test_state_of_torchs_optimizer(kw):
    """A run is taken up from torch.optim.Adam's state_dict, and given back to it."""
    def grads(ps, k):
        for i, p in enumerate(ps):
            p.grad = torch.randn(p.shape, device=DEV, generator=gen(50 * k + i))

    ps, qs = (adam_case([3, 4000], torch.float32, 95, 0)[0] for _ in range(2))
    other, own = torch.optim.Adam(ps, lr=1e-2, **kw), optim.Adam(qs, lr=7.0)
    for k in range(3):
        grads(ps, k)
        other.step()
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    own.load_state_dict(other.state_dict())
    hyper = dict(HYPER, lr=1e-2)
    grads(qs, 3)
    before = snapshot(own, qs, {})
    own.step()
    check_step(own, qs, before, hyper, 4, 1.0)
    back = torch.optim.Adam(ps, lr=5.0, **kw)
    back.load_state_dict(own.state_dict())
    with torch.no_grad():
        for p, q in zip(ps, qs):
            p.copy_(q)
    grads(ps, 4)
    before = [(p.detach().clone(), back.state[p]["exp_avg"].clone(), back.state[p]["exp_avg_sq"].clone()) for p in ps]
    back.step()
    for p, (w, m, v) in zip(ps, before):
        # the other optimizer orders its operations in its own way: a few roundings more
        w1, m1, v1, (ew, em, ev) = adam64(w, p.grad, m, v, 5, 1.0, **hyper)
        assert back.state[p]["step"].item() == 5 and bool(((p.detach().double() - w1).abs() <= 4 * ew).all())


def test_offsets_past_32_bits():
    """Norm, clipping and the step on tensors whose byte and element offsets pass 32 bits."""
    n = 2 ** 32 + 4099
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 4097, n - 1], device=DEV)
    g[at] = torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0, 6.0, 7.0], device=DEV, dtype=torch.bfloat16)
    near(optim.grad_norm([g]), math.sqrt(140.0), 2)
    near(optim.grad_norm([g], math.inf), 7.0, math.inf)
    p = torch.nn.Parameter(g.clone())
    p.grad = g
    near(optim.clip_grad_norm_([p], 1.0), math.sqrt(140.0), 2)
    check_scaled([g[at]], [torch.arange(1.0, 8.0, device=DEV)], 1.0 / (math.sqrt(140.0) + 1e-6))
    opt = optim.Adam([p], lr=0.5)
    opt.step()
    # the first step moves every element with a gradient by lr (to eps and roundings), and no other
    assert int((p.detach() != 0).sum()) == 7
    want = torch.arange(1.0, 8.0, device=DEV) - 0.5
    assert torch.allclose(opt.state[p]["master"][at], want, rtol=1e-5, atol=0)
    del g, p, opt
    torch.cuda.empty_cache()


# --------------------------------------------------------------------------- in the training loop
@pytest.mark.parametrize("limit", [0.05, 0.005])
def test_training_the_network(limit):
    """BPTT steps of the network with folded clipping: each step is the formula's on the network's own
    gradients, and the next forward uses the new weights."""
    from oracle import fixtures as fx
    from v2e2v_amd import CistaLSTCNet
    H, W, C, depth = 16, 16, 32, 2
    torch.manual_seed(0)
    model = CistaLSTCNet([H, W], base_channels=C, depth=depth, num_bins=5).to(DEV).train()
    vox = torch.from_numpy(fx.synthetic_voxels(2, 1, 5, H, W, n_events=200, seed=4)).to(DEV)
    target = torch.rand(1, 1, H, W, device=DEV, generator=gen(1))
    ps = list(model.parameters())
    hyper = dict(HYPER, lr=1e-2)
    opt = make(ps, {}, hyper, max_norm=limit)

    def forward(net):
        prev, state = torch.zeros(1, 1, H, W, device=DEV), None
        for s in range(2):
            prev, state = net(vox[s], prev, state)
        return prev

    for t in (1, 2, 3):
        opt.zero_grad()
        torch.nn.functional.l1_loss(forward(model), target).backward()
        norm = norm64([p.grad for p in ps], 2)
        before = snapshot(opt, ps, {})
        opt.step()
        near(opt.grad_norm, norm, 2)
        check_step(opt, ps, before, hyper, t, min(1.0, limit / (norm + 1e-6)))
        twin = CistaLSTCNet([H, W], base_channels=C, depth=depth, num_bins=5).to(DEV)
        twin.load_state_dict(model.state_dict())
        with torch.no_grad():
            assert torch.equal(forward(model), forward(twin))
