"""Cases of the optimiser operators: the gradient norm with its clip coefficient, AdamW over many tensors with moments in 32 or in
8 bits, and the two together as one optimiser step.

A list of parameters lives in flat buffers here, every tensor at a multiple of 128 elements, so that a pass can hand back its
results whole in a few tensors; the operators themselves are handed the tensors one by one, as views."""
import math
import random

import torch

own = False

BLOCK = 128                    # elements that share one scale of an 8-bit moment
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 5e-4, 0.9, 0.999, 1e-8, 0.01, 1.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTH = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    def c(name, op, **kw):
        d = dict(name=name, op=op, bits=32, kind="networks", copies=1, channels=1, count=0, rows=0, cols=0, param="f32", grad="f32", master=False)
        d.update(kw)
        return d

    return [
        # the trajectory's optimiser: four knots and the camera offset, 30 values - a call's latency
        c("norm trajectory", "norm", kind="pose"),
        # the gradients of one scene's coarse and fine network, 48 tensors, before every step of a run that clips
        c("norm two networks", "norm"),
        # half-precision gradients of a large model, odd row counts
        c("norm large bf16", "norm", kind="matrices", count=5, rows=8191, cols=6400, grad="bf16"),
        # the trajectory again: its own optimiser steps every iteration next to the networks'
        c("adamw32 trajectory", "adamw", kind="pose"),
        # the step of one scene
        c("adamw32 two networks", "adamw"),
        # forty scenes trained in one process: 2000 tensors, most of them biases
        c("adamw32 forty scenes", "adamw", kind="scenes", copies=40, channels=3),
        # half-precision weights with fp32 master copies
        c("adamw32 large bf16 master", "adamw", kind="matrices", count=3, rows=8192, cols=5120, param="bf16", grad="bf16", master=True),
        # the step of one scene with moments in 8 bits
        c("adamw8 two networks", "adamw", bits=8),
        # many weights on one device, where the moments' size is why 8 bits are used
        c("adamw8 large", "adamw", bits=8, kind="matrices", count=4, rows=8192, cols=7168),
        # odd sizes that end inside a block of 128, half-precision weights and gradients
        c("adamw8 ragged bf16", "adamw", bits=8, kind="ragged", count=301, rows=150001, param="bf16", grad="bf16"),
        # what a training loop calls: optimiser.step() with clipping, one scene
        c("step32 two networks", "step"),
        # the same with moments in 8 bits, four colour scenes
        c("step8 four scenes", "step", bits=8, kind="scenes", copies=4, channels=3),
    ]


def draw(rng):
    """Any operator over lists from 30 values to what the largest listed case has, of every type; counts and sizes spread over
    their logarithms."""
    op = rng.choice(("norm", "adamw", "adamw", "step"))
    bits = rng.choice((32, 8))
    kind = rng.choice(("scenes", "matrices", "ragged", "ragged"))
    param, grad, master = rng.choice((("f32", "f32", False), ("f32", "f32", False), ("f32", "bf16", False), ("bf16", "bf16", False), ("bf16", "bf16", True),
                                      ("f16", "f16", False), ("f16", "f32", True)))
    if op == "step" and grad != param:        # a parameter's own gradient has its type
        grad = param
    d = dict(op=op, bits=bits, kind=kind, copies=1, channels=rng.choice((1, 3)), count=0, rows=0, cols=0, param=param, grad=grad, master=master)
    if kind == "scenes":
        d["copies"] = int(round(math.exp(rng.uniform(0.0, math.log(40 if op != "step" else 8)))))
    elif kind == "matrices":
        d["count"] = rng.randint(1, 3)
        d["rows"] = int(round(math.exp(rng.uniform(math.log(16), math.log(8192)))))
        d["cols"] = int(round(math.exp(rng.uniform(math.log(3), math.log(5000)))))
    else:
        d["count"] = int(round(math.exp(rng.uniform(0.0, math.log(400 if op != "step" else 120)))))
        d["rows"] = int(round(math.exp(rng.uniform(math.log(40), math.log(150001)))))
    return d


def _shapes(case):
    """The shapes of the case's list, in order."""
    kind = case["kind"]
    if kind == "pose":
        return [(4, 6), (1, 6)]
    if kind == "matrices":
        return [(case["rows"], case["cols"])] * case["count"]
    if kind == "ragged":                      # sizes from one value up to `rows`, spread over their logarithm; the largest first
        r = random.Random(case["count"] * 1000003 + case["rows"])
        return [(case["rows"],)] + [(max(1, int(case["rows"] ** r.random())),) for _ in range(case["count"] - 1)]
    net = []
    for i in range(8):                        # the 8 x 256 network with the encoding again before its sixth layer
        net += [(256, 63 if i == 0 else 319 if i == 5 else 256), (256,)]
    net += [(128, 283), (128,), (256, 256), (256,), (1, 256), (1,), (case["channels"], 128), (case["channels"],)]
    scene = net + net + ([(4, 6), (1, 6)] if kind == "scenes" else [])
    return scene * case["copies"]


def work(case):
    n = sum(math.prod(s) for s in _shapes(case))
    pw, gw = WIDTH[case["param"]], WIDTH[case["grad"]]
    if case["op"] == "norm":
        return {"bytes": n * gw + 8, "flops": 2 * n}
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    weights = 8 + pw if case["master"] else 2 * pw
    return {"bytes": n * (gw + state + weights), "flops": n * (17 if case["op"] == "step" else 15)}


# ------------------------------------------------------------------------------------------------------------------ inputs
def _slots(case):
    """(offset, shape) of every tensor in the flat buffers, and their length."""
    at, got = 0, []
    for s in _shapes(case):
        got.append((at, s))
        at += -(-math.prod(s) // BLOCK) * BLOCK
    return got, at


def _inputs(case, seed):
    """What both forms and exact() start from, as flat tensors."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(seed)
    slots, n = _slots(case)
    f32 = dict(dtype=torch.float32, device=dev)
    inside = torch.ones(n, **f32)             # 0 in the gaps between two tensors
    size = torch.empty(n, **f32)              # gradients differ in size from tensor to tensor
    how = torch.randn(len(slots), generator=torch.Generator().manual_seed(seed)).tolist()
    for k, (o, s) in enumerate(slots):
        e = o + -(-math.prod(s) // BLOCK) * BLOCK
        inside[o + math.prod(s):e] = 0.0
        size[o:e] = math.exp(1.5 * how[k]) * 1e-3
    size *= inside
    size *= torch.randn(n, generator=gen, **f32).exp_()                  # and from weight to weight
    g = torch.randn(n, generator=gen, **f32).mul_(size)
    g *= torch.rand(n, generator=gen, **f32) > 0.1                       # units that were off send no gradient
    d = {"g": g.to(TYPES[case["grad"]]), "slots": slots, "seed": seed, "t": 100}
    if case["op"] == "norm":
        return d
    master = torch.randn(n, generator=gen, **f32).mul_(0.05).mul_(inside)
    d["p"] = master.to(TYPES[case["param"]])
    if case["master"]:
        d["master"] = master
    m = torch.randn(n, generator=gen, **f32).mul_(size).mul_(0.3)
    u = size * torch.randn(n, generator=gen, **f32).mul_(0.3).exp_()
    if case["bits"] == 32:
        d["m"], d["v"] = m, u * u
    else:
        d["m"], d["ms"] = _nearest(m)
        d["u"], d["us"] = _nearest(u)
    return d


def _power(e):
    """2 ** e for whole e in the range of normal numbers, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _scale(x):
    """The scale of every block of x: a power of two that leaves |x| / scale below 256."""
    top = x.view(-1, BLOCK).abs().amax(1)
    return _power((torch.frexp(top)[1] - 1).clamp_min(-100) - 7)


def _nearest(x):
    """x in 8 bits, as a checkpoint of 32-bit moments is brought in."""
    s = _scale(x)
    return (x.view(-1, BLOCK) / s[:, None]).view(-1).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    d = _inputs(case, seed)
    d["op"], d["bits"] = case["op"], case["bits"]
    if own:
        from benerf_amd import kernels, optim

        def views(name, div=1):
            return [d[name][o // div:o // div + -(-math.prod(s) // div)].view(s if div == 1 else -1) for o, s in d["slots"]] if name in d else None

        g = views("g")
        if case["op"] == "norm":
            d["grads"] = kernels.GradList(g)
            return d
        lists = dict(exp_avg=views("m"), exp_avg_sq=views("v" if case["bits"] == 32 else "u"), exp_avg_scale=views("ms", BLOCK),
                     exp_avg_sq_scale=views("us", BLOCK), master=views("master"))
        if case["op"] == "adamw":
            d["plan"] = kernels.AdamWPlan(views("p"), **lists)
            d["grads"] = kernels.GradList(g, d["plan"])
            return d
        params = [torch.nn.Parameter(p) for p in views("p")]
        opt = optim.FusedAdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"], max_norm=MAX_NORM,
                               master=case["master"], seed=seed)
        for k, p in enumerate(params):
            opt.state[p] = dict({name: v[k] for name, v in lists.items() if v is not None}, step=torch.tensor(float(d["t"])))
            p.grad = g[k]
        d["opt"] = opt
    return d


# ------------------------------------------------------------------------------------------------------------------ a pass
def run(d):
    if own:
        return _run_own(d)
    out = {}
    gs = None
    if d["op"] != "adamw":
        norm = d["g"].double().square().sum().sqrt()
        coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        out["norm"] = torch.stack((norm, coef)).float()
        if d["op"] == "norm":
            return out
        gs = out["norm"][1]
    d["t"] += 1
    t = d["t"]
    g = d["g"].float()
    if gs is not None:
        g = g * gs
    p = d["master"] if "master" in d else d["p"].float()
    if d["bits"] == 32:
        m, v = d["m"], d["v"]
    else:
        m = (d["m"].float().view(-1, BLOCK) * d["ms"][:, None]).view(-1)
        v = (d["u"].float().view(-1, BLOCK) * d["us"][:, None]).view(-1).square()
    m = m + (g - m) * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    root = v.sqrt()
    p = p * (1 - LR * DECAY)
    p = p - LR / (1 - BETA1 ** t) * (m / (root / math.sqrt(1 - BETA2 ** t) + EPS))
    if "master" in d:
        d["master"].copy_(p)
        out["master"] = d["master"]
    d["p"].copy_(p)
    out["p"] = d["p"]
    if d["bits"] == 32:
        out["m"], out["v"] = d["m"].copy_(m), d["v"].copy_(v)
        return out
    low, high = _halves(m.numel(), d["seed"], t, m.device)
    for name, scale, x, h in (("m", "ms", m, low), ("u", "us", root, high)):
        s = _scale(x)
        y = (x.view(-1, BLOCK) / s[:, None]).view(-1)
        step = _power((torch.frexp(y.abs())[1] - 1).clamp_min(-6) - 3)
        q = (y.abs() / step + h.float() / 65536).floor() * step
        if name == "u":
            q = torch.where(x > 0, q.clamp_min(2.0 ** -9), q)
        out[name], out[scale] = d[name].copy_(torch.copysign(q, y)), d[scale].copy_(s)
    return out


def _halves(n, seed, t, dev):
    """The two 16-bit draws of every element: Philox4x32-10 over groups of four, counter (group, t), key = seed."""
    c = torch.arange(n // 4, dtype=torch.int64, device=dev)
    low32 = 0xFFFFFFFF
    x, y = c & low32, c >> 32
    z, w = torch.full_like(c, t), torch.full_like(c, 0x40000000)
    k0, k1 = seed & low32, seed >> 32 & low32

    def turn(x, y, z, w, k0, k1):
        a, b = x * 0xD2511F53, z * 0xCD9E8D57
        return (b >> 32 & low32) ^ y ^ k0, b & low32, (a >> 32 & low32) ^ w ^ k1, a & low32

    for r in range(10):
        x, y, z, w = turn(x, y, z, w, k0 + r * 0x9E3779B9 & low32, k1 + r * 0xBB67AE85 & low32)
    h = torch.stack((x, y, z, w), 1).view(-1)
    return h & 0xFFFF, h >> 16


def _run_own(d):
    from benerf_amd import kernels

    if d["op"] == "norm":
        return {"norm": kernels.grad_norm(d["grads"], max_norm=MAX_NORM)[:2]}
    if d["op"] == "adamw":
        d["t"] += 1
        kernels.adamw_step(d["plan"], d["grads"], lr=LR, step=d["t"], betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, seed=d["seed"])
        return {k: d[k] for k in ("master", "p", "m", "v", "ms", "u", "us") if k in d}
    d["opt"].step()
    return dict({k: d[k] for k in ("master", "p", "m", "v", "ms", "u", "us") if k in d}, norm=d["opt"].grad_norm[:2])


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The first pass over these inputs, from the definitions, in 64 bits and in pieces of the list."""
    d = _inputs(case, seed)
    out, coef = {}, 1.0
    n = d["g"].numel()
    pieces = [(a, min(a + (1 << 26), n)) for a in range(0, n, 1 << 26)]
    if case["op"] != "adamw":
        total = math.fsum(float(torch.linalg.vector_norm(d["g"][a:b].double())) ** 2 for a, b in pieces)
        coef = min(1.0, MAX_NORM / (math.sqrt(total) + 1e-6))
        out["norm"] = torch.tensor([math.sqrt(total), coef], dtype=torch.float64)
        if case["op"] == "norm":
            return out
    t = d["t"] + 1
    parts = {}
    for a, b in pieces:
        g = d["g"][a:b].double() * coef
        p = (d["master"] if case["master"] else d["p"])[a:b].double()
        if case["bits"] == 32:
            m, v = d["m"][a:b].double(), d["v"][a:b].double()
        else:
            m, u = (d[q][a:b].double() * d[s][a // BLOCK:b // BLOCK].double().repeat_interleave(BLOCK) for q, s in (("m", "ms"), ("u", "us")))
            v = u ** 2
        m, v = BETA1 * m + (1 - BETA1) * g, BETA2 * v + (1 - BETA2) * g ** 2
        new = (1 - LR * DECAY) * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
        got = {"p": new, "m": m, "v": v}
        if case["bits"] == 8:
            del got["v"]
            words = _philox(torch.arange(a // 4, b // 4, dtype=torch.int64, device=g.device), t, seed)
            for name, x, r in (("m", m, words % 65536), ("u", v.sqrt(), words // 65536)):
                top = x.abs().reshape(-1, BLOCK).max(1).values
                s = 2.0 ** (torch.where(top > 0, torch.floor(torch.log2(top.clamp_min(1e-300))), -1000.0).clamp_min(-100.0) - 7.0)
                y = x.abs() / s.repeat_interleave(BLOCK)
                ulp = 2.0 ** (torch.floor(torch.log2(y.clamp_min(1e-300))).clamp_min(-6.0) - 3.0)
                q = ulp * torch.floor(y / ulp + r.double() / 65536.0)
                if name == "u":
                    q = torch.where((y > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
                got[name] = q * torch.sign(x)
        if case["master"]:
            got["master"] = new
        for k, x in got.items():
            parts.setdefault(k, []).append(x)
    out.update({k: torch.cat(x) for k, x in parts.items()})
    if case["bits"] == 8:                     # a scale jumps by two where a block's largest value is next to a power of two
        out["ms"] = out["us"] = None
    return out


def _philox(c, t, seed):
    """Four words for every counter, written from the generator's definition: per round two products, their halves crossed."""
    m32 = (1 << 32) - 1
    v = [c % (1 << 32), c // (1 << 32), torch.full_like(c, t), torch.full_like(c, 1 << 30)]
    key = [seed % (1 << 32), seed // (1 << 32)]
    for _ in range(10):
        lo0, lo1 = (v[0] * 0xD2511F53) & m32, (v[2] * 0xCD9E8D57) & m32
        hi0, hi1 = ((v[0] * 0xD2511F53) >> 32) & m32, ((v[2] * 0xCD9E8D57) >> 32) & m32
        v = [hi1 ^ v[1] ^ key[0], lo1, hi0 ^ v[3] ^ key[1], lo0]
        key = [(key[0] + 0x9E3779B9) & m32, (key[1] + 0xBB67AE85) & m32]
    return torch.stack(v, dim=1).reshape(-1)
