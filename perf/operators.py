"""Cases of the training-step operators: gradient norm, gradient clipping, Adam step.

All three work on many tensors at once.  In every case the tensors are views of one flat buffer,
as gradients are after a backward pass of the network (its gradient buffer, each parameter in a
slot of 64 elements) or after data-parallel averaging in buckets (tensors end to end, at odd
offsets).  The plain forms below use that: they are whole-buffer operations, with no loop over
the tensors.  The slots' padding holds zeros, which no operator changes.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST = 300_000_000          # elements of the largest drawn case; the listed ones reach more bytes


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # the gradients of the default network (base_channels 64, 25 tensors, 1.4 M): watched every step
        dict(name="norm_c64", op="norm", sizes="net", channels=64, type="f32", p="2"),
        # many bf16 tensors end to end, 1.2 GB: a large model's gradients
        dict(name="norm_bf16_large", op="norm", sizes="ragged", tensors=320, total=600_000_011, layout=1, type="bf16", p="2"),
        # the largest gradient, float16, a middling model with odd sizes
        dict(name="norm_max_f16", op="norm", sizes="ragged", tensors=97, total=24_000_007, layout=2, type="f16", p="inf"),
        # clipping of the default network's gradients, norm over the limit
        dict(name="clip_c64", op="clip", sizes="net", channels=64, type="f32", p="2", limit=0.3),
        # the widest network that trains (base_channels 256, 22 M), norm within the limit: nothing changes
        dict(name="clip_inside_c256", op="clip", sizes="net", channels=256, type="f32", p="2", limit=3.0),
        # bf16 gradients, 211 tensors of odd sizes, norm over the limit
        dict(name="clip_bf16_ragged", op="clip", sizes="ragged", tensors=211, total=150_000_001, layout=3, type="bf16", p="2", limit=0.1),
        # fine-tuning of the biases alone: the smallest step, where latency counts
        dict(name="adam_biases", op="adam", sizes="biases", channels=64, type="f32", t=17, decay=0.0, decoupled=False, clip=False, p="2", limit=1.0),
        # the training script's step: default network, no clipping, no decay
        dict(name="adam_c64", op="adam", sizes="net", channels=64, type="f32", t=1000, decay=0.0, decoupled=False, clip=False, p="2", limit=1.0),
        # the same with clipping folded in
        dict(name="adam_c64_clip", op="adam", sizes="net", channels=64, type="f32", t=1000, decay=0.0, decoupled=False, clip=True, p="2", limit=0.3),
        # the widest network, early in training, decay in the gradient, clipping by the largest value
        dict(name="adam_c256_decay", op="adam", sizes="net", channels=256, type="f32", t=1, decay=0.01, decoupled=False, clip=True, p="inf", limit=0.5),
        # a large model in float32, decoupled decay, clipping: bandwidth counts
        dict(name="adamw_f32_large", op="adam", sizes="ragged", tensors=147, total=268_000_003, layout=4, type="f32", t=20000, decay=0.05, decoupled=True, clip=True, p="2", limit=0.2),
        # a large model in bf16 with float32 master weights, many tensors of odd sizes
        dict(name="adamw_bf16_large", op="adam", sizes="ragged", tensors=301, total=200_000_033, layout=5, type="bf16", t=300, decay=0.1, decoupled=True, clip=True, p="2", limit=0.2),
    ]


def draw(rng):
    op = rng.choice(["norm", "clip", "adam"])
    case = dict(op=op, type=rng.choice(["f32", "f32", "bf16", "f16"]), p=rng.choice(["2", "2", "2", "1", "inf"]))
    if rng.random() < 0.35:
        case.update(sizes=rng.choice(["net", "net", "biases"]), channels=32 * rng.randint(1, 8))
    else:
        total = int(math.exp(rng.uniform(math.log(100), math.log(MOST))))
        most = max(1, min(400, total // 10))
        case.update(sizes="ragged", tensors=int(math.exp(rng.uniform(0, math.log(most)))) if most > 1 else 1,
                    total=total, layout=rng.randint(10, 1 << 20))
    if op != "norm":
        case["limit"] = round(math.exp(rng.uniform(math.log(0.05), math.log(2.0))), 3)
    if op == "adam":
        case.update(t=rng.choice([0, 1, 9, 100, 5000, 100000]), decay=rng.choice([0.0, 0.01, 0.1]),
                    decoupled=rng.random() < 0.5, clip=rng.random() < 0.6)
    return case


def _sizes(case):
    """Elements of each tensor, and the multiple that each one's place in the flat buffer is rounded up to."""
    if case["sizes"] == "ragged":
        r, n, total = random.Random(case["layout"]), case["tensors"], case["total"]
        w = [math.exp(r.uniform(0, 7)) for _ in range(n)]
        got = [max(1, int(total * x / sum(w))) for x in w]
        got[got.index(max(got))] += total - sum(got)
        return got, 1
    C, h = case["channels"], case["channels"] // 2
    net = [(h, 5), (h, 1), (C, C), (4 * C, 3 * C), (2 * C, 4 * C), (2 * C, C), None,
           (C, 2 * C), (2 * C, C), (C, 2 * C), (4 * C, 2 * C), (C, C), (1, C)]
    biases = [s[0] for s in net if s]
    if case["sizes"] == "biases":
        return biases, 64
    return [n for s in net for n in ((2 * C,) if s is None else (9 * s[0] * s[1], s[0]))], 64


# ------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    sizes, slot = _sizes(case)
    at, end = [], 0
    for n in sizes:
        at.append(end)
        end += n + (-n % slot)
    kind, dev = TYPES[case["type"]], "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    used = torch.zeros(end, device=dev)
    for a, n in zip(at, sizes):
        used[a:a + n] = 1.0
    # gradients: a scale of its own for each tensor, the norm about 1 (p = 2)
    pick = random.Random(seed)
    fresh = torch.randn(end, device=dev, generator=gen) * used
    for a, n in zip(at, sizes):
        fresh[a:a + n] *= math.exp(pick.uniform(-1.5, 1.5))
    unit = {"2": lambda g: g.double().square().sum().sqrt(), "1": lambda g: g.double().abs().sum(),
            "inf": lambda g: g.abs().max()}[case["p"]](fresh)
    # in float16 a norm of 1 over many elements would leave denormals: the loss is scaled there
    fresh = (fresh * (1.0 / unit.float()) * pick.uniform(0.7, 1.4) * (256.0 if case["type"] == "f16" else 1.0)).to(kind)
    state = dict(case=case, sizes=sizes, fresh=fresh)
    grads = fresh if case["op"] != "clip" else torch.empty_like(fresh)
    if case["op"] == "clip":
        grads.copy_(fresh)
    state["flat"] = grads
    state["grads"] = [grads[a:a + n] for a, n in zip(at, sizes)]
    state["limit"] = case.get("limit", 1.0) * (256.0 if case["type"] == "f16" else 1.0)
    if case["op"] == "norm":
        return state
    master = torch.randn(end, device=dev, generator=gen).mul_(0.05).mul_(used)
    params = master if kind == torch.float32 else master.to(kind)
    state["params"] = [torch.nn.Parameter(params[a:a + n]) for a, n in zip(at, sizes)]
    for p, g in zip(state["params"], state["grads"]):
        p.grad = g
    if case["op"] == "clip":
        return state
    # moments of a run that has come to step t (none before the first)
    started = 1.0 if case["t"] else 0.0
    rms = 1.0 / math.sqrt(sum(sizes)) * (256.0 if case["type"] == "f16" else 1.0)
    state["exp_avg"] = torch.randn(end, device=dev, generator=gen).mul_(0.3 * rms * started).mul_(used)
    state["exp_avg_sq"] = torch.rand(end, device=dev, generator=gen).mul_(rms * rms * started).mul_(used)
    state["steps"] = torch.full((len(sizes),), float(case["t"]), device=dev)
    state.update(t=case["t"], weights=params, master=master)
    state["slots"] = {p: dict(step=state["steps"][i], exp_avg=state["exp_avg"][a:a + n], exp_avg_sq=state["exp_avg_sq"][a:a + n],
                              **({} if kind == torch.float32 else {"master": master[a:a + n]}))
                      for i, (p, a, n) in enumerate(zip(state["params"], at, sizes))}
    return state


LR, BETAS, EPS = 1e-4, (0.9, 0.999), 1e-8


# ------------------------------------------------------------------------- plain forms
def _plain_norm(flat, p):
    g = flat.float()
    if p == "inf":
        return g.abs().max()
    if p == "1":
        return g.abs().sum()
    return g.square().sum().sqrt()


def _plain_scale(norm, limit):
    return (limit / (norm + 1e-6)).clamp(max=1.0)


def _plain(state):
    case, flat = state["case"], state["flat"]
    if case["op"] == "norm":
        return {"norm": _plain_norm(flat, case["p"])}
    if case["op"] == "clip":
        flat.copy_(state["fresh"])
        norm = _plain_norm(flat, case["p"])
        flat.copy_(flat.float() * _plain_scale(norm, state["limit"]))
        return {"grads": flat, "norm": norm}
    w, m, v, (b1, b2) = state["master"], state["exp_avg"], state["exp_avg_sq"], BETAS
    g, out = flat.float(), {}
    if case["clip"]:
        out["norm"] = _plain_norm(flat, case["p"])
        g = g * _plain_scale(out["norm"], state["limit"])
    if case["decoupled"]:
        w.mul_(1.0 - LR * case["decay"])
    elif case["decay"]:
        g = g + w * case["decay"]
    state["t"] += 1
    state["steps"].add_(1.0)
    m.mul_(b1).add_(g, alpha=1.0 - b1)
    v.mul_(b2).addcmul_(g, g, value=1.0 - b2)
    root = v.sqrt().mul_(1.0 / math.sqrt(1.0 - b2 ** state["t"])).add_(EPS)
    w.sub_((m / root).mul_(LR / (1.0 - b1 ** state["t"])))
    if state["weights"] is not w:
        state["weights"].copy_(w)
    return dict(out, **_updated(state))


def _updated(state):
    got = dict(weights=state["weights"], exp_avg=state["exp_avg"], exp_avg_sq=state["exp_avg_sq"], steps=state["steps"])
    if state["weights"] is not state["master"]:
        got["master"] = state["master"]
    return got


# -------------------------------------------------------------- the framework's operators
def _own(state):
    from v2e2v_amd import optim
    case = state["case"]
    p = float(case["p"])
    if case["op"] == "norm":
        return {"norm": optim.grad_norm(state["grads"], p)}
    if case["op"] == "clip":
        state["flat"].copy_(state["fresh"])      # the gradients that a backward pass writes anew for each step
        norm = optim.clip_grad_norm_(state["params"], state["limit"], norm_type=p)
        return {"grads": state["flat"], "norm": norm}
    opt = state.get("optimizer")
    if opt is None:                              # a run that is taken up again at step t
        opt = optim.Adam(state["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=case["decay"],
                         decoupled_weight_decay=case["decoupled"], max_norm=state["limit"] if case["clip"] else None,
                         norm_type=p)
        opt.state.update(state["slots"])
        state["optimizer"] = opt
    opt.step()
    return dict({"norm": opt.grad_norm} if case["clip"] else {}, **_updated(state))


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------- work, exact values
def work(case):
    n = sum(_sizes(case)[0])
    s = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        return {"bytes": n * s, "flops": 2 * n}
    if case["op"] == "clip":                     # the fresh gradients read, the clipped ones written
        return {"bytes": 2 * n * s, "flops": 3 * n}
    # gradient, weight and both moments read; weight and moments written (a 16-bit weight is written from its master copy)
    return {"bytes": n * 28, "flops": n * (16 + (3 if case["clip"] else 0))}


def exact(case, seed):
    s = prepare(case, seed)
    x = s["fresh"].to(torch.float64)
    order = float(case["p"])
    norm = x.abs().amax() if order == math.inf else torch.pow(torch.pow(x.abs(), order).sum(), 1.0 / order)
    shrink = torch.ones_like(norm)
    if case["op"] == "clip" or case.get("clip"):
        shrink = torch.minimum(shrink, s["limit"] / (norm + 1e-6))
    if case["op"] == "norm":
        return {"norm": norm}
    x *= shrink
    if case["op"] == "clip":
        return {"grads": x, "norm": norm}
    w = s["master"].to(torch.float64)
    if not case["decoupled"]:
        x += case["decay"] * w
    t, (b1, b2) = case["t"] + 1, BETAS
    m = s["exp_avg"].to(torch.float64)
    m += (1.0 - b1) * (x - m)
    v = s["exp_avg_sq"].to(torch.float64)
    v += (1.0 - b2) * (x * x - v)
    if case["decoupled"]:
        w = w - LR * case["decay"] * w
    w = w - LR * (m / (1.0 - b1 ** t)) / ((v / (1.0 - b2 ** t)).sqrt() + EPS)
    got = dict(weights=w, exp_avg=m, exp_avg_sq=v, steps=s["steps"].to(torch.float64) + 1.0)
    if s["weights"] is not s["master"]:
        got["master"] = w
    if case["clip"]:
        got["norm"] = norm
    return got
