"""GPU: optim.FusedAdamW - torch.optim.AdamW over K9 - against torch's own AdamW in float64, with the calls a training program makes:
groups, missing gradients, checkpoints in either form, moved parameters, clipping, capture, hooks."""
import copy
import io

import numpy as np
import pytest
import torch

import adamw_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def optim():
    from benerf_amd import optim
    return optim


def _params(sizes=((64, 63), (64,), (1, 64), (1,), (3, 5, 7)), dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.1).to(dtype).cuda()) for s in sizes]


def _twins(params):
    return [torch.nn.Parameter(p.detach().double().cpu()) for p in params]


def _grads(params, twins, seed, absent=()):
    gen = torch.Generator().manual_seed(1000 + seed)
    for k, (p, t) in enumerate(zip(params, twins)):
        g = (torch.randn(p.shape, generator=gen) * 0.02 * (k + 1)).to(p.dtype)
        p.grad = None if k in absent else g.cuda()
        t.grad = None if k in absent else g.double()


def _close(params, twins, steps, lr, extra=0.0):
    # a step's error is at most 3 u |p| + 19 u lr (oracle/adamw_oracle.py: |update| <= a few lr here, dm / den below 8 u |update| / 0.1);
    # 200 u lr a step leaves room for the accumulated moments
    for p, t in zip(params, twins):
        d = (p.detach().double().cpu() - t.detach()).abs()
        assert float((d - steps * (4 * O.HALF * t.detach().abs() + 200 * O.HALF * lr) - extra).max()) <= 0, float(d.max())


def test_equals_torch_adamw(optim):
    """Two groups with their own rates and decay, rates changed between the steps, a parameter that misses gradients for two steps, one
    added later: values and step counts as torch's AdamW in float64."""
    ps = _params()
    ts = _twins(ps)
    groups = lambda q: [dict(params=q[:2], lr=1e-2, weight_decay=0.1), dict(params=q[2:], lr=1e-3, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.0)]      # noqa: E731
    ours, ref = optim.FusedAdamW(groups(ps)), torch.optim.AdamW(groups(ts))
    assert isinstance(ours, torch.optim.AdamW)
    late, late_t = _params([(17,)], seed=7), None
    for it in range(8):
        if it == 5:
            late_t = _twins(late)
            ours.add_param_group(dict(params=late, lr=2e-3))
            ref.add_param_group(dict(params=late_t, lr=2e-3))
        _grads(ps, ts, it, absent=(1, 3) if it in (2, 3) else ())
        if late_t:
            _grads(late, late_t, 50 + it)
        for o in (ours, ref):
            for g in o.param_groups:
                g["lr"] *= 0.9
            o.step()
    _close(ps + late, ts + late_t, 8, 1e-2)
    for p, t in zip(ps + late, ts + late_t):
        assert float(ours.state[p]["step"]) == float(ref.state[t]["step"])
        m, v = ours.state[p]["exp_avg"].double().cpu(), ours.state[p]["exp_avg_sq"].double().cpu()
        rm, rv = ref.state[t]["exp_avg"], ref.state[t]["exp_avg_sq"]
        assert float((m - rm).abs().max()) <= 64 * O.HALF * float(rm.abs().max() + 0.1) and float(((v - rv).abs() / (rv + 1e-30)).max()) <= 100 * O.HALF


def test_clipping_equals_torch(optim):
    ps = _params()
    ts = _twins(ps)
    ours, ref = optim.FusedAdamW([dict(params=ps[:3]), dict(params=ps[3:], lr=3e-3)], max_norm=0.3), torch.optim.AdamW([dict(params=ts[:3]), dict(params=ts[3:], lr=3e-3)])
    for it in range(6):
        _grads(ps, ts, it)
        total = float(torch.nn.utils.clip_grad_norm_(ts, 0.3))
        before = [p.grad.clone() for p in ps]
        ours.step()
        ref.step()
        assert abs(float(ours.grad_norm[0]) - total) <= 4 * O.HALF * total and total > 0.3
        assert all(torch.equal(p.grad, b) for p, b in zip(ps, before)), "gradients are not rewritten"
    _close(ps, ts, 6, 3e-3)
    # a step that is not finite leaves everything, and its count
    snap = [p.detach().clone() for p in ps]
    _grads(ps, ts, 9)
    ps[0].grad[0, 0] = float("inf")
    ours.step()
    assert all(torch.equal(p, s) for p, s in zip(ps, snap)) and float(ours.grad_norm[2]) == 1.0 and float(ours.state[ps[0]]["step"]) == 6.0
    _grads(ps, ts, 9)
    torch.nn.utils.clip_grad_norm_(ts, 0.3)
    ours.step()
    ref.step()
    _close(ps, ts, 7, 3e-3)
    assert float(ours.grad_norm[3]) == 1.0 and float(ours.state[ps[0]]["step"]) == 7.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_master_copies_keep_small_updates(optim, dtype):
    """Updates far below a half-precision step: lost without float32 copies, kept with them."""
    sizes = [(1000,), (33,)]
    plain, kept = _params(sizes, dtype), _params(sizes, dtype)
    ts = [torch.nn.Parameter(p.detach().double().cpu()) for p in kept]
    a = optim.FusedAdamW(plain, lr=1e-6, weight_decay=0.0)
    b = optim.FusedAdamW(kept, lr=1e-6, weight_decay=0.0, master=True)
    ref = torch.optim.AdamW(ts, lr=1e-6, weight_decay=0.0)
    start = [p.detach().clone() for p in plain]
    for it in range(20):
        _grads(kept, ts, 0)
        for p, q in zip(plain, kept):
            p.grad = q.grad.clone()
        for o in (a, b, ref):
            o.step()
    for k, (q, t) in enumerate(zip(kept, ts)):
        master = b.state[q]["master"].double().cpu()
        assert float((master - t.detach()).abs().max()) <= 20 * (4 * O.HALF * float(t.abs().max()) + 200 * O.HALF * 1e-6)
        assert torch.equal(q.detach(), b.state[q]["master"].to(dtype))
    big = start[0].abs() > 0.05
    assert torch.equal(plain[0].detach()[big], start[0][big])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpoint_round_trip(optim, bits, dtype):
    """state_dict through torch.save (tensors only) into a new optimiser: the next steps are the same bits, whatever the parameter's type."""
    master = dtype != torch.float32
    make = lambda ps: optim.FusedAdamW([dict(params=ps[:2]), dict(params=ps[2:], lr=5e-4)], state_bits=bits, master=master, max_norm=1.0, seed=5)      # noqa: E731
    ps = _params(dtype=dtype)
    a = make(ps)
    for it in range(3):
        _grads(ps, _twins(ps), it)
        a.step()
    f = io.BytesIO()
    torch.save({"o": a.state_dict(), "p": [p.detach() for p in ps]}, f)
    f.seek(0)
    ck = torch.load(f, weights_only=True)
    qs = [torch.nn.Parameter(x) for x in ck["p"]]
    b = make(qs)
    b.load_state_dict(ck["o"])
    for it in range(3, 6):
        for group in (ps, qs):
            _grads(group, _twins(group), it)
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        assert set(a.state[p]) == set(b.state[q])
        for k in a.state[p]:
            x, y = a.state[p][k], b.state[q][k]
            assert x.dtype == y.dtype and torch.equal(x.cpu().reshape(-1).view(torch.uint8), y.cpu().reshape(-1).view(torch.uint8)), k
    assert (a.state[ps[0]]["exp_avg"].dtype == torch.float8_e4m3fn) == (bits == 8)


def test_checkpoints_between_forms(optim):
    """torch's AdamW -> 8 bits -> 32 bits -> torch's AdamW: step counts exact, moments as far off as a rounding to nearest."""
    ps = _params()
    ref = torch.optim.AdamW(ps, lr=1e-3)
    for it in range(4):
        _grads(ps, _twins(ps), it)
        ref.step()
    eight = optim.FusedAdamW(ps, lr=1e-3, state_bits=8)
    eight.load_state_dict(copy.deepcopy(ref.state_dict()))
    for p in ps:
        p.grad = torch.zeros_like(p)
    keep = [p.detach().clone() for p in ps]
    eight.step()
    assert float(eight.state[ps[0]]["step"]) == 5.0 and eight.state[ps[0]]["exp_avg"].dtype == torch.float8_e4m3fn
    for p, k in zip(ps, keep):
        p.data.copy_(k)
    wide = optim.FusedAdamW(ps, lr=1e-3)
    wide.load_state_dict(copy.deepcopy(eight.state_dict()))
    wide.step()
    for p in ps:
        m = ref.state[p]["exp_avg"].double() * 0.9 ** 2
        # to nearest (2^-4), once more at random (2^-3), or 2^-9 of 256 below the range
        d = (wide.state[p]["exp_avg"].double() - m).abs()
        assert bool((d <= 0.2 * m.abs() + 2.0 ** -15 * m.abs().max()).all())
        v = ref.state[p]["exp_avg_sq"].double() * 0.999 ** 2
        assert bool(((wide.state[p]["exp_avg_sq"].double() - v).abs() <= 0.45 * v + 2.0 ** -28 * v.max()).all())
    back = torch.optim.AdamW(ps, lr=1e-3)
    back.load_state_dict(wide.state_dict())
    back.step()
    assert float(back.state[ps[0]]["step"]) == 7.0


def test_moved_parameters_and_assigned_state_are_followed(optim):
    ps = _params()
    ts = _twins(ps)
    ours, ref = optim.FusedAdamW(ps, lr=1e-2), torch.optim.AdamW(ts, lr=1e-2)
    for it in range(6):
        if it == 2:
            old = ps[0].data
            ps[0].data = ps[0].data.clone()
            old.fill_(7.0)
        if it == 4:
            for o, q in ((ours, ps[2]), (ref, ts[2])):
                o.state[q]["exp_avg"] = torch.zeros_like(q)
                o.state[q]["exp_avg_sq"] = torch.zeros_like(q)
                o.state[q]["step"] = torch.tensor(0.0)
            o2 = {k: v.clone() if torch.is_tensor(v) else v for k, v in ours.state[ps[1]].items()}
            ours.state[ps[1]] = o2
        _grads(ps, ts, it)
        if it == 3:                       # a gradient with strides of its own
            ps[0].grad = ps[0].grad.t().contiguous().t()
            ps[4].grad = torch.ones(3, 1, 1, device="cuda").expand(3, 5, 7)
            ts[4].grad = torch.ones(3, 5, 7, dtype=torch.float64)
        ours.step()
        ref.step()
    _close(ps, ts, 6, 1e-2)
    assert float(ours.state[ps[2]]["step"]) == 2.0 and float(ours.state[ps[1]]["step"]) == 6.0
    ps[3].data = torch.zeros(9, device="cuda")
    with pytest.raises((RuntimeError, ValueError)):
        ours.step()


def test_closure_hooks_deepcopy_and_refusals(optim):
    ps = _params([(4,)])
    o = optim.FusedAdamW(ps, lr=0.1, weight_decay=0.0)
    calls = []

    def closure():
        o.zero_grad()
        loss = (ps[0] ** 2).sum()
        loss.backward()
        return loss
    o.register_step_pre_hook(lambda *a: calls.append("pre"))
    o.register_step_post_hook(lambda *a: calls.append("post"))
    for _ in range(31):
        want = float((ps[0].detach() ** 2).sum())
        assert float(o.step(closure)) == want
    assert calls[:2] == ["pre", "post"] and len(calls) == 62
    sched = torch.optim.lr_scheduler.StepLR(o, 1, 0.5)
    o.step(closure)
    sched.step()
    assert o.param_groups[0]["lr"] == 0.05
    twin = copy.deepcopy(o)
    assert twin.state_bits == 32 and len(twin.state) == 1
    empty = optim.FusedAdamW([torch.nn.Parameter(torch.zeros(3, device="cuda"))])
    assert empty.step() is None and len(empty.state) <= 1
    sp = torch.nn.Parameter(torch.zeros(3, 3, device="cuda"))
    so = optim.FusedAdamW([sp])
    sp.grad = torch.eye(3, device="cuda").to_sparse()
    with pytest.raises((NotImplementedError, RuntimeError)):
        so.step()
    shared = torch.zeros(8, device="cuda")
    with pytest.raises(ValueError):
        two = [torch.nn.Parameter(shared[:5]), torch.nn.Parameter(shared[3:])]
        bad = optim.FusedAdamW(two)
        for p in two:
            p.grad = torch.ones_like(p)
        bad.step()
    strided = torch.nn.Parameter(torch.zeros(6, 4, device="cuda").t())
    strided.grad = torch.ones_like(strided)
    with pytest.raises(ValueError):
        optim.FusedAdamW([strided]).step()


def test_under_a_gradient_scaler(optim):
    """Factors that are powers of two change nothing; a gradient that overflowed skips the step, its moments and its counter."""
    plain, scaled = _params([(40, 5), (3,)]), _params([(40, 5), (3,)])
    a, b = optim.FusedAdamW(plain, max_norm=0.5), optim.FusedAdamW(scaled, max_norm=0.5)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=1000)
    x = torch.randn(16, 40, generator=torch.Generator().manual_seed(1)).cuda()

    def loss(ps, factor=1.0):
        return ((x @ ps[0]).square().mean() + ps[1].square().sum()) * factor
    for it in range(5):
        if it == 2:
            before = [p.detach().clone() for p in scaled]
            scaler.scale(loss(scaled, 1e38)).backward()
            scaler.step(b)
            scaler.update()
            b.zero_grad()
            assert all(torch.equal(p, q) for p, q in zip(scaled, before)) and scaler.get_scale() == 512.0 and float(b.state[scaled[0]]["step"]) == 2.0
        loss(plain).backward()
        a.step()
        a.zero_grad()
        scaler.scale(loss(scaled)).backward()
        scaler.step(b)
        scaler.update()
        b.zero_grad()
        assert all(torch.equal(p, q) for p, q in zip(plain, scaled))


@pytest.mark.parametrize("bits,clip", [(32, None), (8, 0.2)])
def test_captured_optimiser_step(optim, bits, clip):
    """capturable: backward and step in one graph, replayed next to eager work; equal to an eager twin, counters on the device."""
    def build():
        ps = _params([(64, 64), (64,), (1,)], seed=3)
        return ps, optim.FusedAdamW(ps, lr=1e-3, state_bits=bits, max_norm=clip, capturable=True, seed=9)
    (pa, a), (pb, b) = build(), build()
    x = torch.randn(32, 64, device="cuda")

    def once(ps, o, x):
        o.zero_grad(set_to_none=True)
        loss = ((torch.tanh(x @ ps[0] + ps[1]) * ps[2]) ** 2).mean()
        loss.backward()
        o.step()
        return loss.detach()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            once(pa, a, x)
            once(pb, b, x)
    torch.cuda.current_stream().wait_stream(side)
    xs = x.clone()
    g = torch.cuda.CUDAGraph()
    a.zero_grad(set_to_none=True)
    with torch.cuda.graph(g):
        la = once(pa, a, xs)
    for it in range(4):
        x = torch.randn(32, 64, device="cuda")
        xs.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        lb = once(pb, b, x)
        assert float(la) == float(lb)
        for p, q in zip(pa, pb):
            assert torch.equal(p, q)
    assert float(a.state[pa[0]]["step"]) == 6.0
    c = optim.FusedAdamW(_params([(4,)]), lr=1e-3)
    c.param_groups[0]["params"][0].grad = torch.ones(4, device="cuda")
    c.step()
    h = torch.cuda.CUDAGraph()
    error = None
    with torch.cuda.graph(h):
        torch.zeros(1, device="cuda")
        try:
            c.step()
        except RuntimeError as e:
            error = str(e)
    assert error and "counter" in error and float(c.state[c.param_groups[0]["params"][0]]["step"]) == 1.0


@pytest.mark.parametrize("bits", [32, 8])
def test_what_a_capture_may_not_begin_with(optim, bits):
    """A first step, or the first one that misses a gradient, inside a capture: refused, and nothing of the optimiser is left half-made."""
    ps = _params([(40,), (9,)])
    o = optim.FusedAdamW(ps, lr=1e-3, state_bits=bits, max_norm=1.0, capturable=True)

    def refused(absent):
        errors = []
        for k, p in enumerate(ps):
            p.grad = None if k in absent else torch.ones_like(p)
        torch.cuda.synchronize()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.zeros(1, device="cuda")
            try:
                o.step()
            except RuntimeError as e:
                errors.append(str(e))
        return errors
    before = [p.detach().clone() for p in ps]
    assert "outside" in refused(())[0] and not any(o.state.values()) and o.grad_norm is None
    o.step()
    assert "missing" in refused((1,))[0]
    assert float(o.state[ps[0]]["step"]) == 1.0 and float(o.state[ps[1]]["step"]) == 1.0
    for p in ps:
        p.grad = torch.ones_like(p)
    o.step()
    assert all(float(o.state[p]["step"]) == 2.0 for p in ps) and not torch.equal(before[0], ps[0])


def test_rates_as_tensors_and_settings_that_change(optim):
    ps = _params([(50,)])
    ts = _twins(ps)
    lr = torch.tensor(1e-2)
    o, ref = optim.FusedAdamW(ps, lr=lr), torch.optim.AdamW(ts, lr=1e-2)
    for it in range(4):
        if it == 2:
            o.param_groups[0]["capturable"] = True          # counters move to the device, with their values
            o.param_groups[0]["lr"] = torch.tensor(1e-2, device="cuda")
        _grads(ps, ts, it)
        o.step()
        ref.step()
    _close(ps, ts, 4, 1e-2, extra=4 * 1e-2 * 2.0 ** -24)
    assert o.state[ps[0]]["step"].is_cuda and float(o.state[ps[0]]["step"]) == 4.0


def test_eight_bits_train_like_thirty_two(optim):
    """The expectation of the stored moments is the moment: over many steps with gradients of constant size the mean of sqrt(v) follows
    its 32-bit value, where rounding to nearest would have stood still at the first step's."""
    n, steps = 128 * 64, 400
    size = torch.logspace(-4, 0, 128, device="cuda").repeat(64)
    wide, eight = [torch.nn.Parameter(torch.zeros(n, device="cuda")) for _ in range(2)]
    a, b = optim.FusedAdamW([wide], lr=1e-3, weight_decay=0.0), optim.FusedAdamW([eight], lr=1e-3, weight_decay=0.0, state_bits=8, seed=2)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(steps):
        g = torch.randn(n, device="cuda", generator=gen) * size
        wide.grad, eight.grad = g, g.clone()
        a.step()
        b.step()
    u = a.state[wide]["exp_avg_sq"].sqrt().view(64, 128).mean(0)
    st = b.state[eight]
    q = optim.decode_moment(st["exp_avg_sq"], st["exp_avg_sq_scale"]).view(64, 128)
    # sqrt(v) wanders by the roundings of the last 1 / (1 - b2) steps; its mean over 64 elements by an eighth of that
    ratio = (q.mean(0) / u).double()
    assert 0.9 <= float(ratio.mean()) <= 1.1 and float((ratio - 1).abs().max()) <= 0.35
    # and so the weights: same displacement up to the noise of the rates
    dw, de = wide.detach().view(64, 128).std(0), eight.detach().view(64, 128).std(0)
    assert 0.85 <= float((de / dw).mean()) <= 1.15


def test_seeds_and_groups_draw_apart(optim):
    ps = _params([(4096,), (4096,)])
    with torch.no_grad():
        ps[1].copy_(ps[0])
    o = optim.FusedAdamW([dict(params=ps[:1]), dict(params=ps[1:])], state_bits=8, seed=1)
    for _ in range(2):
        g = torch.randn(4096, device="cuda")
        for p in ps:
            p.grad = g.clone()
        o.step()
    a, b = (o.state[p]["exp_avg"].view(torch.uint8) for p in ps)
    assert not torch.equal(a, b)


def test_flat_adam_still_refuses_decay(optim):
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    p.grad = torch.ones_like(p)
    with pytest.raises(NotImplementedError):
        optim.FlatAdam([p], weight_decay=0.1).step()
