"""GPU: the optimiser operators over lists (K9) against a 64-bit evaluation (oracle/adamw_oracle.py): gradient norm with clip coefficient
and verdict, AdamW with moments in 32 and 8 bits.  The bounds are the oracle's, counted in roundings; a rounding to bfloat16 is 2^-8 of the
value, to float16 2^-11 (2^-25 below its normal range)."""
import gc
import math

import numpy as np
import pytest
import torch

import adamw_oracle as O

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
GUARD = 37                      # elements on both sides of a tensor that nobody may touch


@pytest.fixture(scope="module")
def K():
    from benerf_amd import kernels
    return kernels


def _f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def _narrow(x, kind):
    """A rounding of float64 values to `kind`, at most."""
    return {"f32": 0.0, "bf16": 2.0 ** -8 * np.abs(x), "f16": 2.0 ** -11 * np.abs(x) + 2.0 ** -25}[kind]


class Buffers:
    """Tensors inside larger ones, at odd offsets, with known values around them."""

    def __init__(self):
        self.held = []

    def put(self, x, shift=0):
        x = x.cuda()
        raw = x.element_size() == 1                       # float8 knows no fill
        whole = torch.full((x.numel() + 2 * GUARD + shift,), 91 if raw else 0.25, dtype=torch.uint8 if raw else x.dtype, device="cuda")
        a = GUARD + shift
        view = whole[a:a + x.numel()]
        view.copy_(x.reshape(-1).view(torch.uint8) if raw else x.reshape(-1))
        self.held.append((whole, a, x.numel()))
        return (view.view(x.dtype) if raw else view).view(x.shape)

    def check(self):
        for whole, a, n in self.held:
            want = 91 if whole.dtype == torch.uint8 else 0.25
            assert bool((whole[:a] == want).all()) and bool((whole[a + n:] == want).all()), "written outside a tensor"


class List:
    """A list of parameters, gradients and moments with its oracle."""

    def __init__(self, K, sizes, param="f32", grad="f32", bits=32, master=False, seed=0, shift=0, t=5, zero=False):
        gen = torch.Generator().manual_seed(seed + 1)
        rand = lambda n: torch.randn(n, generator=gen)      # noqa: E731
        self.K, self.sizes, self.bits, self.param, self.buf = K, sizes, bits, param, Buffers()
        put = lambda x: self.buf.put(x, shift)              # noqa: E731
        from benerf_amd import optim
        self.p, self.g, self.m, self.v, self.ms, self.vs, self.master = [], [], [], [], [], [], []
        for k, n in enumerate(sizes):
            size = 10.0 ** (k % 5 - 4) * torch.exp(rand(n))
            w = rand(n) * 0.1
            g = rand(n) * size * (torch.rand(n, generator=gen) > 0.1)
            m, u = rand(n) * size * 0.3, size * torch.exp(0.3 * rand(n))
            if zero:
                m, u = torch.zeros(n), torch.zeros(n)
            self.p.append(put(w.to(TYPES[param])))
            self.g.append(put(g.to(TYPES[grad])))
            if master:
                self.master.append(put(w))
            if bits == 32:
                self.m.append(put(m))
                self.v.append(put(u * u))
            else:
                for x, code, scale in ((m, self.m, self.ms), (u, self.v, self.vs)):
                    c, s = optim.encode_moment(x)
                    code.append(put(c))
                    scale.append(put(torch.zeros_like(s) if zero else s))
        kw = dict(exp_avg_scale=self.ms, exp_avg_sq_scale=self.vs) if bits == 8 else {}
        self.plan = K.AdamWPlan(self.p, self.m, self.v, master=self.master or None, **kw)
        self.t, self.seed = t, seed

    def state(self, k):
        """(weight, gradient, m, v) of tensor k in float64."""
        if self.bits == 32:
            m, v = _f64(self.m[k]), _f64(self.v[k])
        else:
            rep = lambda s: np.repeat(_f64(s), 128)[:self.sizes[k]]      # noqa: E731
            m, v = _f64(self.m[k]) * rep(self.ms[k]), (_f64(self.v[k]) * rep(self.vs[k])) ** 2
        return _f64(self.master[k] if self.master else self.p[k]), _f64(self.g[k]), m, v

    def snapshot(self):
        return [self.state(k) for k in range(len(self.sizes))]

    def check(self, before, scale=1.0, t=None, hyper=HYPER, absent=()):
        """Every tensor against one oracle step from `before`."""
        t = self.t if t is None else t
        block = 0
        for k, n in enumerate(self.sizes):
            p, g, m, v = before[k]
            after = self.state(k)
            if k in absent:
                assert all(np.array_equal(a, b) for a, b in zip(before[k], after)), "tensor %d was to be left alone" % k
                block += -(-n // 128)
                continue
            (p2, m2, v2), (dp, dm, dv, du) = O.step(p, g, m, v, hyper["lr"], t, hyper["betas"], hyper["eps"], hyper["weight_decay"], scale)
            got = after[0]
            if self.master:
                assert np.all(np.abs(got - p2) <= dp), ("master", k, n)
                assert np.all(np.abs(_f64(self.p[k]) - got) <= _narrow(got, self.param)), ("rounded master", k, n)
            else:
                assert np.all(np.abs(got - p2) <= dp + _narrow(np.abs(p2) + dp, self.param)), ("p", k, n, np.max(np.abs(got - p2) - dp))
            if self.bits == 32:
                assert np.all(np.abs(after[2] - m2) <= dm) and np.all(np.abs(after[3] - v2) <= dv), ("moments", k, n)
            else:
                low, high = O.draws(n, block, t, self.seed)
                for name, x, dx, r, codes, scales, keep in (("m", m2, dm, low, self.m[k], self.ms[k], False), ("u", np.sqrt(v2), du, high, self.v[k], self.vs[k], True)):
                    val = np.abs(_f64(codes) * np.repeat(_f64(scales), 128)[:n])
                    lo, hi = O.coded_range(x, dx, r, keep)
                    assert np.all((lo <= val) & (val <= hi)), (name, k, n, int(((lo > val) | (val > hi)).sum()))
                    sc = _f64(scales)
                    ok = (sc >= O.scale_of(np.maximum(np.abs(x) - dx, 0))) & (sc <= O.scale_of(np.abs(x) + dx))
                    assert np.all(ok), (name + " scale", k, n)
                sign = np.sign(_f64(self.m[k]))
                assert np.all((sign == 0) | (sign == np.sign(m2)) | (np.abs(m2) <= dm)), ("sign of m", k)
            block += -(-n // 128)
        self.buf.check()


SIZES = [1, 2, 3, 4, 5, 127, 128, 129, 0, 255, 1000, 1023, 1024, 1025, 4097, 20000]
COMBOS = [("f32", "f32", False), ("f32", "bf16", False), ("f32", "f16", False), ("bf16", "bf16", False), ("bf16", "f32", True), ("bf16", "bf16", True),
          ("bf16", "f16", False), ("f16", "f16", False), ("f16", "f32", False), ("f16", "f16", True), ("f16", "bf16", True)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad,master", COMBOS)
def test_step_against_64_bits(K, param, grad, master, bits):
    """Two steps over a list of all the odd sizes, one tensor without a gradient, at offsets that only an element's alignment holds."""
    for shift in (0, 1):
        L = List(K, SIZES, param, grad, bits, master, seed=11 + shift, shift=shift)
        for _ in range(2):
            before = L.snapshot()
            grads = [None if k == 10 else g for k, g in enumerate(L.g)]
            K.adamw_step(L.plan, grads, step=L.t, seed=L.seed, guard_range=False, **HYPER)
            L.check(before, absent=(10,))
            L.t += 1


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_from_zero_moments(K, bits):
    """t = 1, moments (and 8-bit scales) of zero: |update| = lr for every gradient that is not negligible; zero gradients move nothing but decay."""
    L = List(K, SIZES, bits=bits, t=1, zero=True)
    before = L.snapshot()
    K.adamw_step(L.plan, L.g, step=1, seed=L.seed, **HYPER)
    L.check(before)
    for k in range(len(SIZES)):
        p, g = before[k][0], before[k][1]
        now = _f64(L.p[k])
        assert np.allclose(now[g == 0], p[g == 0] * (1 - HYPER["lr"] * HYPER["weight_decay"]), rtol=1e-6, atol=0)
        if bits == 8:
            u = _f64(L.v[k])
            assert np.array_equal(u > 0, g != 0), "a second moment was rounded to zero, or made from nothing"


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [63, 64, 65, 480, 481, 1100])
def test_long_lists(K, bits, count):
    """More tensors than one launch carries; gradients missing at the edges of launches."""
    sizes = [1 + (37 * k) % 300 for k in range(count)]
    L = List(K, sizes, bits=bits, seed=count)
    before = L.snapshot()
    absent = {0, count - 1, 62, 479 if count > 479 else 5}
    K.adamw_step(L.plan, [None if k in absent else g for k, g in enumerate(L.g)], step=L.t, seed=L.seed, **HYPER)
    L.check(before, absent=absent)
    words = K.grad_norm(K.GradList(L.g), 1.0)
    norm, coef = O.clip_words([_f64(g) for g in L.g], 1.0)
    assert abs(float(words[0]) - norm) <= 2 * O.HALF * norm and abs(float(words[1]) - coef) <= 2 * O.HALF * coef


@pytest.mark.parametrize("bits", [32, 8])
def test_a_large_tensor_next_to_small_ones(K, bits):
    """Thousands of chunks, so that runs of 64 go to one XCD each; the last one partial."""
    L = List(K, [3, 2200001, 129, 4096, 100003], bits=bits, seed=5)
    before = L.snapshot()
    K.adamw_step(L.plan, L.g, step=L.t, seed=L.seed, **HYPER)
    L.check(before)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_norm_against_64_bits(K, kind):
    gen = torch.Generator().manual_seed(2)
    for sizes in ([1], [0, 1, 0], SIZES, [2200001, 5]):
        buf = Buffers()
        g = [buf.put((torch.randn(n, generator=gen) * 0.3).to(TYPES[kind]), shift=1) for n in sizes]
        for max_norm, gs in ((1.0, 1.0), (1e6, 0.125), (float("inf"), -2.0)):
            words = K.grad_norm(g, max_norm, gs).tolist()
            norm, coef = O.clip_words([_f64(x) for x in g], max_norm, gs)
            # sums in 64 bits, one rounding to 32: 2^-24, doubled for the root's own
            assert abs(words[0] - norm) <= 2 * O.HALF * norm and abs(words[1] - coef) <= 2 * O.HALF * coef and words[2:] == [0.0, 0.0]
        buf.check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[512 * 32], [512 * 32 + 1], [511] * 32, [511] * 33, [1] * 64, [513] * 16, [512 * 31, 1, 1]])
def test_norm_of_short_lists(K, sizes, kind):
    """Around the 32 chunks of 512 that one workgroup takes: all gradients, without the last, the first or those between, counted on the device."""
    gen = torch.Generator().manual_seed(len(sizes))
    buf = Buffers()
    g = [buf.put((torch.randn(n, generator=gen) * 0.3).to(TYPES[kind]), shift=1) for n in sizes]
    words, steps = torch.zeros(4, device="cuda"), [torch.zeros(1, device="cuda") for _ in range(64)]
    absent = ([], [len(g) - 1], [0], range(1, len(g) - 1))
    for it, none in enumerate(absent):
        here = [None if k in none and len(g) > 1 else x for k, x in enumerate(g)]
        K.grad_norm(here, 0.5, -2.0, out=words, counters=steps)
        norm, coef = O.clip_words([_f64(x) for x in here if x is not None], 0.5, -2.0)
        got = words.tolist()
        assert abs(got[0] - norm) <= 2 * O.HALF * norm and abs(got[1] - coef) <= 2 * O.HALF * coef and got[2:] == [0.0, 0.0]
        assert all(float(s) == it + 1 for s in steps)
    buf.check()


def test_norm_range_and_verdict(K):
    """Squares beyond f32's range both ways; inf and NaN are a verdict; the count of skipped steps goes on in the caller's words."""
    big, small = torch.full((1000,), 1e30, device="cuda"), torch.full((1000,), 1e-30, device="cuda")
    assert abs(float(K.grad_norm([big])[0]) / (1e30 * math.sqrt(1000)) - 1) <= 4 * O.HALF
    assert abs(float(K.grad_norm([small])[0]) / (1e-30 * math.sqrt(1000)) - 1) <= 4 * O.HALF
    words = torch.zeros(4, device="cuda")
    steps = [torch.zeros(1, device="cuda"), torch.full((), 7.0, device="cuda")]
    n_skip = 0
    for bad in (None, float("nan"), float("inf"), -float("inf"), None):
        g = torch.randn(5000, device="cuda")
        if bad is not None:
            g[4711] = bad
            n_skip += 1
        K.grad_norm([small, g], 1.0, out=words, counters=steps)
        assert words[2].item() == (bad is not None) and words[3].item() == n_skip
        assert bad is None or words[1].item() == 0.0
    assert float(steps[0]) == 2.0 and float(steps[1]) == 9.0
    empty = K.grad_norm(K.GradList([torch.empty(0, device="cuda"), None]), 1.0).tolist()
    assert empty == [0.0, 1.0, 0.0, 0.0]


@pytest.mark.parametrize("bits", [32, 8])
def test_norm_and_step_together(K, bits):
    """The run of them: clipped steps, one of them skipped for a NaN and not counted, several lists under one norm."""
    A, B = List(K, [300, 5000, 1], "bf16", "bf16", bits, True, seed=3, t=1), List(K, [77, 129], bits=bits, seed=4, t=1)
    words = torch.zeros(4, device="cuda")
    applied = 0
    for it in range(4):
        keep = A.g[1].clone()
        if it == 2:
            A.g[1][17] = float("nan")
        before = A.snapshot(), B.snapshot()
        K.grad_norm([K.GradList(A.g, A.plan), K.GradList(B.g, B.plan)], 0.05, grad_scale=0.5, out=words)
        for L in (A, B):
            K.adamw_step(L.plan, L.g, step=it + 1, grad_scale=0.5, norm=words, seed=L.seed, **HYPER)
        if it == 2:
            for L, b in zip((A, B), before):
                assert all(np.array_equal(x, y, equal_nan=True) for s, r in zip(b, L.snapshot()) for x, y in zip(s, r)), "a skipped step wrote something"
            A.g[1].copy_(keep)
            continue
        applied += 1
        _, coef = O.clip_words([_f64(g) for g in A.g + B.g], 0.05, 0.5)
        assert coef < 1.0
        for L, b in zip((A, B), before):
            L.check(b, scale=0.5 * coef, t=applied)
    assert words[3].item() == 1.0


def test_guard_words_skip_and_count(K):
    """The MLP range guard's words, as adam_step reads them: a violation skips the step, skipped ones are not counted."""
    from benerf_amd import _lib
    L = List(K, [500], t=4)
    st = torch.zeros(_lib.ST_WORDS, dtype=torch.int32, device="cuda")
    st[_lib.ST_SKIP] = 1
    before = L.snapshot()
    K.adamw_step(L.plan, L.g, step=6, status=st, **HYPER)
    assert all(np.array_equal(a, b) for a, b in zip(before[0], L.state(0)))
    words = K.grad_norm(L.g, 1.0, guard_range=True, status=st)
    assert words[2].item() == 1.0
    count = torch.zeros(1, device="cuda")
    K.adamw_count(count, status=st)
    assert count.item() == 0.0
    st[_lib.ST_SKIP] = 0
    st[_lib.ST_SKIPPED_TOTAL] = 2
    K.adamw_step(L.plan, L.g, step=6, status=st, **HYPER)
    L.check(before, t=4)
    K.adamw_count(count, status=st)
    assert count.item() == 1.0
    # with a norm its count is the only one: steps that the guard skipped are in it once
    words = torch.zeros(4, device="cuda")
    L = List(K, [500], t=4)
    for it in range(6):
        st[_lib.ST_SKIP] = int(it in (1, 2))
        st[_lib.ST_SKIPPED_TOTAL] += int(it in (1, 2))
        before = L.snapshot()
        K.grad_norm(L.g, float("inf"), out=words, status=st)
        K.adamw_step(L.plan, L.g, step=it + 1, norm=words, status=st, **HYPER)
        if it in (1, 2):
            assert all(np.array_equal(a, b) for a, b in zip(before[0], L.state(0)))
        else:
            L.check(before, t=it + 1 - int(it > 1) - int(it > 2))


@pytest.mark.parametrize("bits", [32, 8])
def test_non_finite_values_stay_with_themselves(K, bits):
    """Without a norm, inf and NaN gradients poison their own element and no other - in 8 bits neither its block's codes nor scale."""
    L = List(K, [1000], bits=bits, seed=9)
    L.g[0][3], L.g[0][130], L.g[0][999] = float("nan"), float("inf"), -float("inf")
    clean = L.g[0].clone()
    bad = ~clean.isfinite()
    before = L.snapshot()
    K.adamw_step(L.plan, L.g, step=L.t, seed=L.seed, **HYPER)
    assert bool(L.p[0][bad].isnan().all()) and bool(L.p[0][~bad].isfinite().all())
    b = bad.cpu().numpy()
    (p2, m2, v2), (dp, dm, dv, du) = O.step(before[0][0], np.where(b, 0.0, before[0][1]), *before[0][2:], HYPER["lr"], L.t, HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
    assert np.all(np.abs(_f64(L.p[0]) - p2)[~b] <= dp[~b])
    if bits == 8:
        assert bool(L.m[0].float()[bad].isnan().all()) and bool(L.m[0].float()[~bad].isfinite().all())
        x = np.where(b, np.nan, m2)
        sc = _f64(L.ms[0])
        assert np.all((sc >= O.scale_of(np.abs(x) - dm)) & (sc <= O.scale_of(np.abs(x) + dm)))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-8, 1e-15])
def test_values_at_the_ends_of_the_range(K, bits, eps):
    """Gradients whose squares are denormal or vanish, next to ordinary ones and alone in their block; large ones below the square's end."""
    L = List(K, [640], bits=bits, seed=13, t=1, zero=True)
    g = L.g[0]
    g[0:128] *= 0
    g[5] = 3e-20                       # alone: its square is denormal
    g[128:256] = torch.logspace(-25, -17, 128, device="cuda")
    g[256:384] = torch.logspace(-20, 0, 128, device="cuda")
    g[384:512] = torch.logspace(10, 18, 128, device="cuda")
    hyper = dict(HYPER, eps=eps)
    for t in (1, 2, 3):
        before = L.snapshot()
        K.adamw_step(L.plan, L.g, step=t, seed=L.seed, **hyper)
        L.check(before, t=t, hyper=hyper)
    assert bool(L.p[0].isfinite().all())


@pytest.mark.parametrize("bits", [32, 8])
def test_counter_and_rate_on_the_device(K, bits):
    L = List(K, [1000, 7], bits=bits, seed=21, t=1)
    step, lr = torch.zeros((), device="cuda"), torch.tensor([HYPER["lr"]], device="cuda")
    for t in (1, 2, 3):
        before = L.snapshot()
        K.adamw_count(step, guard_range=False)
        K.adamw_step(L.plan, L.g, step=step, seed=L.seed, **dict(HYPER, lr=lr))
        # the learning rate is a float32 here
        L.check(before, t=t, hyper=dict(HYPER, lr=float(lr)))
    far = torch.full((), 1.0e6, device="cuda")
    before = L.snapshot()
    K.adamw_step(L.plan, L.g, step=far, seed=L.seed, **HYPER)
    L.check(before, t=1000000)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(K, bits):
    """Norm, clip and step in a graph, replayed with other gradients in place and eager work in between: each replay equals the eager
    step of a twin; a captured step without a device counter is refused."""
    A, B = List(K, SIZES, bits=bits, seed=31, t=1), List(K, SIZES, bits=bits, seed=31, t=1)

    def once(L, step, words, grads):
        K.grad_norm(grads, 0.02, out=words, counters=[step])
        K.adamw_step(L.plan, grads, step=step, norm=words, seed=L.seed, **HYPER)

    sets = [(L, torch.zeros((), device="cuda"), torch.zeros(4, device="cuda"), K.GradList(L.g, L.plan)) for L in (A, B)]
    for s in sets:
        once(*s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once(*sets[0])
    for it in range(5):
        noise = torch.randn(20000, device="cuda") * (1.0 if it != 2 else float("nan"))
        for L in (A, B):
            L.g[-1].copy_(noise)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.randn(1000, 1000, device="cuda") @ torch.randn(1000, 1000, device="cuda")
        once(*sets[1])
        assert float(eager.sum()) == float(eager.sum())
        for x, y in zip(A.p + A.m + A.v + A.ms + A.vs, B.p + B.m + B.v + B.ms + B.vs):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), it
        assert torch.equal(sets[0][1], sets[1][1]) and torch.equal(sets[0][2].view(torch.int32), sets[1][2].view(torch.int32))
    assert float(sets[0][1]) == 5.0 and float(sets[0][2][3]) == 1.0
    from benerf_amd import _lib
    refused = []
    side = torch.cuda.CUDAGraph()
    with torch.cuda.graph(side):
        torch.zeros(1, device="cuda")
        for call in (lambda: K.adamw_step(A.plan, sets[0][3], step=3, **HYPER), lambda: K.AdamWPlan(A.p, A.m, A.v), lambda: K.grad_norm(A.g)):
            try:
                call()
            except (_lib.BenerfHipError, ValueError) as e:
                refused.append(str(e))
    assert len(refused) == 3 and "counter" in refused[0] and "captured region" in refused[-1]


def test_another_stream_and_the_plan_let_go(K):
    """Launches go to the current stream; a plan dropped while its launch is queued on another stream stays valid for it."""
    side = torch.cuda.Stream()
    for it in range(3):
        L = List(K, [200000, 33], seed=it)
        before = L.snapshot()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            busy = torch.randn(4096, 4096, device="cuda")
            for _ in range(4):
                busy = busy @ busy * 1e-2
            K.adamw_step(L.plan, L.g, step=L.t, **HYPER)
        del L.plan
        torch.full((4096,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        L.check(before)


def test_a_captured_step_outlives_its_plan(K):
    """A graph reads the plan's table at every replay, also after the caller has let plan and lists go."""
    L = List(K, [3000, 33], seed=8, t=1)
    step, words = torch.zeros((), device="cuda"), torch.zeros(4, device="cuda")
    lists = [K.GradList(L.g, L.plan), K.GradList(L.g)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.grad_norm(lists[1], 0.02, out=words, counters=[step])
        K.adamw_step(L.plan, lists[0], step=step, norm=words, **HYPER)
    tables = [part.dev_at for x in (L.plan, lists[1]) for part in x.parts]
    assert all(at in K._captured for at in tables)
    before = L.snapshot()
    del L.plan, lists
    gc.collect()
    filled = [torch.full((256 << k,), 255, dtype=torch.uint8, device="cuda") for k in range(8) for _ in range(8)]
    assert not any(x.data_ptr() in tables for x in filled)
    _, coef = O.clip_words([_f64(g) for g in L.g], 0.02, 1.0)
    for t in (1, 2, 3):
        graph.replay()
        torch.cuda.synchronize()
        L.check(before, scale=coef, t=t)
        before = L.snapshot()
    assert float(step) == 3.0


@pytest.mark.parametrize("sizes", [[300, 7], [200000, 33], [1000] * 70])
def test_norms_at_once(K, sizes):
    """Two graphs over one list, replayed on two streams beside an eager call on a third: nobody's sums reach another's words."""
    gen = torch.Generator().manual_seed(4)
    g = [torch.randn(n, generator=gen).cuda() for n in sizes]
    grads = K.GradList(g)
    want = [O.clip_words([_f64(x) for x in g], 1.0, scale)[0] for scale in (1.0, 2.0, 3.0)]
    K.grad_norm(grads)
    graphs, words = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [torch.zeros(4, device="cuda") for _ in range(3)]
    for graph, w, scale in zip(graphs, words, (1.0, 2.0)):
        with torch.cuda.graph(graph):
            K.grad_norm(grads, 1.0, scale, out=w)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for it in range(4):
        for w in words:
            w.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for stream, graph in zip(streams, graphs):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(streams[2]):
                K.grad_norm(grads, 1.0, 3.0, out=words[2])
        torch.cuda.synchronize()
        for w, norm in zip(words, want):
            assert abs(float(w[0]) - norm) <= 2 * O.HALF * norm and w[2:].tolist() == [0.0, 0.0]


def test_same_result_every_time(K):
    """No order of atomics, no leftover: the same inputs give the same bits, seeds give other roundings."""
    def once(seed):
        L = List(K, [50000, 129], bits=8, seed=1)
        w = K.grad_norm(L.g, 0.1)
        K.adamw_step(L.plan, L.g, step=3, norm=w, seed=seed, **HYPER)
        return [x.view(torch.uint8).clone() for x in L.p + L.m + L.v + [w]]
    a, b, c = once(1), once(1), once(2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(a[0], c[0]) and not torch.equal(a[2], c[2])


def test_refusals_on_the_device(K):
    f = lambda n, d=torch.float32: torch.zeros(n, dtype=d, device="cuda")      # noqa: E731
    p, m, v = [f(8), f(5)], [f(8), f(5)], [f(8), f(5)]
    plan = K.AdamWPlan(p, m, v)
    same = f(8)
    for args, kw in ((([f(8), f(8)[::2]], m, v), {}), ((p, [f(8), f(4)], v), {}), ((p, [f(8)], v), {}), (([same, same], [f(8), f(8)], [f(8), f(8)]), {}),
                     ((p, m, m), {}), ((p, m, v), dict(exp_avg_scale=[f(1), f(1)])), ((p, m, v), dict(master=p)),
                     (([f(8, torch.bfloat16)], [f(8)], [f(8)]), dict(master=[f(7)])),
                     ((p, [x.to(K.CODE_TYPE) for x in m], [x.to(K.CODE_TYPE) for x in v]), {}),
                     ((p, [x.to(K.CODE_TYPE) for x in m], [x.to(K.CODE_TYPE) for x in v]), dict(exp_avg_scale=[f(1), f(2)], exp_avg_sq_scale=[f(1), f(1)]))):
        with pytest.raises(ValueError):
            K.AdamWPlan(*args, **kw)
    for args in (([f(8, torch.float64), f(5)], m, v), (p, [f(8, torch.bfloat16), f(5)], v), (p, [f(8, torch.bfloat16)] * 2, v), ([f(8), 3.0], m, v)):
        with pytest.raises(TypeError):
            K.AdamWPlan(*args)
    with pytest.raises(TypeError):
        K.adamw_step(plan, [f(8, torch.float64), f(5)], 1e-3, 1)
    for bad in ([f(8)], [f(8), f(6)], [f(8), f(10)[::2]], K.GradList([f(8), f(6)])):
        with pytest.raises(ValueError):
            K.adamw_step(plan, bad, 1e-3, 1)
    g = [f(8), f(5)]
    for kw in (dict(step=0), dict(step=1, betas=(1.0, 0.9)), dict(step=1, eps=-1.0), dict(step=1, weight_decay=-0.1)):
        from benerf_amd import _lib
        with pytest.raises(_lib.BenerfHipError):
            K.adamw_step(plan, g, 1e-3, **kw)
    word = lambda n, d=torch.int32, **kw: torch.zeros(n, dtype=d, **dict(dict(device="cuda"), **kw))      # noqa: E731
    for kw in (dict(step=f(2)), dict(step=torch.zeros(1)), dict(step=1, norm=f(3)), dict(step=1, status=word(15)), dict(step=1, status=word(16, device="cpu"))):
        with pytest.raises(ValueError):
            K.adamw_step(plan, g, 1e-3, **kw)
    for call in (lambda **kw: K.grad_norm(g, 1.0, **kw), lambda **kw: K.adamw_count(f(1), **kw)):
        for kw, error in ((dict(status=word(15)), ValueError), (dict(status=word(16, device="cpu")), ValueError), (dict(status=word(16, torch.float32)), TypeError)):
            with pytest.raises(error):
                call(**kw)
    with pytest.raises(ValueError):
        K.grad_norm(g, 1.0, out=f(3))
    with pytest.raises(TypeError):
        K.adamw_step(plan, g, 1e-3, f(1, torch.float64))
    assert not any(bool(x.any()) for x in p + m + v)


def test_parameter_updates_reach_the_packed_networks(K):
    """The step writes through addresses: packed copies of network weights have to notice."""
    L = List(K, [100])
    gen = K._param_generation
    K.adamw_step(L.plan, L.g, step=1, **HYPER)
    assert K._param_generation > gen


@pytest.mark.parametrize("bits", [8, 32])
def test_offsets_beyond_32_bits(K, bits):
    """One bfloat16 tensor of more than 2^32 elements: the ends and the places where 31 and 32 bits run over, against the oracle."""
    n = (1 << 32) + 1003
    need = n * (2 + 2 + (2 if bits == 8 else 8)) + (4 << 30)
    if torch.cuda.mem_get_info()[0] < need:
        pytest.skip("needs %.0f GiB of free device memory" % (need / 2 ** 30))
    p, g = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    kind = torch.uint8 if bits == 8 else torch.float32
    m, v = torch.zeros(n, dtype=kind, device="cuda"), torch.zeros(n, dtype=kind, device="cuda")
    kw = {}
    if bits == 8:
        m, v = m.view(K.CODE_TYPE), v.view(K.CODE_TYPE)
        kw = {name: [torch.zeros(-(-n // 128), device="cuda")] for name in ("exp_avg_scale", "exp_avg_sq_scale")}
    spans = [(0, 256), ((1 << 31) - 128, (1 << 31) + 128), ((1 << 32) - 128, (1 << 32) + 128), (n - 107, n)]
    for a, b in spans:
        g[a:b] = torch.randn(b - a, device="cuda").to(torch.bfloat16)
    gs = [_f64(g[a:b]) for a, b in spans]
    plan = K.AdamWPlan([p], [m], [v], **kw)
    words = K.grad_norm([g], 1.0)
    norm, coef = O.clip_words(gs, 1.0)
    assert abs(float(words[0]) - norm) <= 2 * O.HALF * norm
    K.adamw_step(plan, [g], step=1, norm=words, seed=6, **HYPER)
    for (a, b), x in zip(spans, gs):
        (p2, m2, v2), (dp, dm, dv, du) = O.step(np.full(b - a, 0.5), x, np.zeros(b - a), np.zeros(b - a), HYPER["lr"], 1, HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], coef)
        assert np.all(np.abs(_f64(p[a:b]) - p2) <= dp + 2.0 ** -8 * (np.abs(p2) + dp))
        if bits == 8:
            low, high = (r[a % 4:] for r in O.draws(b - a + a % 4, a // 128, 1, 6))
            scale = lambda name: np.repeat(_f64(kw[name][0][a // 128:-(-b // 128)]), 128)[a % 128:a % 128 + b - a]      # noqa: E731
            if a % 128 == 0:
                for x2, dx, r, c, name, keep in ((m2, dm, low, m, "exp_avg_scale", False), (np.sqrt(v2), du, high, v, "exp_avg_sq_scale", True)):
                    lo, hi = O.coded_range(x2, dx, r, keep)
                    val = np.abs(_f64(c[a:b]) * scale(name))
                    assert np.all((lo <= val) & (val <= hi)), (name, a)
        else:
            assert np.all(np.abs(_f64(m[a:b]) - m2) <= dm) and np.all(np.abs(_f64(v[a:b]) - v2) <= dv)
    quiet = p[1000:(1 << 31) - 200]
    assert bool((quiet == quiet[0]).all())
