"""GPU: optimiser state between forms and owners - checkpoints of one networks' optimiser resumed with another."""
import numpy as np
import pytest
import torch

import adamw_oracle as O
from test_adamw_paths_gpu import _run, _setting
from test_api_gpu import DEV, _graph

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["adam", "adamw"])
def test_eight_bit_checkpoint_resumed_in_32_bits(tmp_path, kind):
    """A run with adamw8, saved, loaded into the objects of another networks' optimiser and into its TrainStep: the moments are the values that
    the codes stand for, and the next step is the formula's from them."""
    from benerf_amd import checkpoint as CK, engine, optim
    args, cam, HW, accu, img = _setting(benerf_optimizer="adamw8", benerf_weight_decay=0.0)
    model_a, g_a = _graph(args, seed=3)
    a = engine.TrainStep(g_a, args, cam, cam, torch.device(DEV), seed=21)
    _run(a, HW, accu, img, 0, 3)
    optims = model_a.setup_optimizer(args)
    a.export_optimizer_state(optims)
    path = str(tmp_path / "ck.tar")
    CK.save(path, g_a, optims, a.global_step)
    n = 2 * a.n_net
    args_b = _setting(benerf_optimizer=kind, benerf_weight_decay=0.0)[0]
    model_b, g_b = _graph(args_b, seed=8)
    ob = model_b.setup_optimizer(args_b)
    b = engine.TrainStep(g_b, args_b, cam, cam, torch.device(DEV), seed=21)
    b.import_optimizer_state(ob, CK.load(path, g_b, ob))
    assert torch.equal(a.flat_p, b.flat_p)
    for k, x in enumerate(a.net_plan.params):
        held = optim.convert_moments({name: ts[k] for name, ts in a.net_moments.items()}, 32)
        at = slice(x.storage_offset(), x.storage_offset() + x.numel())
        assert torch.equal(b.flat_m[at], held["exp_avg"].reshape(-1)) and torch.equal(b.flat_v[at], held["exp_avg_sq"].reshape(-1)), k
    p, m, v = (f[:n].double().cpu().numpy() for f in (b.flat_p, b.flat_m, b.flat_v))
    lr = b._lr(args.lrate, args.decay_rate)
    _run(b, HW, accu, img, 3, 4)
    (p2, _, _), (dp, _, _, _) = O.step(p, b.flat_g[:n].double().cpu().numpy(), m, v, lr, 4, (0.9, 0.999), 1e-8, 0.0)
    # the oracle's bound holds for either formula's order: both have one product, root, sum and quotient, Adam's kernel a division in place of a product
    # by a rounded constant (a rounding less)
    worst = abs(b.flat_p[:n].double().cpu().numpy() - p2) - dp
    assert worst.max() <= 0, worst.max()


def f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def _one_step(p, g, m, v, lr, t, got, master, rounding):
    """got and master, if there is one, against the oracle's step (decay 0.01)."""
    (p2, m2, v2), (dp, _, _, _) = O.step(p, g, m, v, lr, t, (0.9, 0.999), 1e-8, 0.01)
    if master is not None:
        assert (abs(master - p2) - dp).max() <= 0
        p2, dp = master, 0.0
    assert (abs(got - p2) - dp - rounding * (abs(p2) + dp)).max() <= 0
    return m2, v2


@pytest.mark.parametrize("dtype,half", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_weights_loaded_after_a_step(dtype, half):
    """Weights loaded in place, their masters dropped: the next step starts from the loaded weights, and the state has masters again.  A master that
    is assigned is the one that the step reads."""
    from benerf_amd import optim
    gen = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen)      # noqa: E731
    ps = [torch.nn.Parameter((rand(40, 33) + 3).to(dtype).cuda()), torch.nn.Parameter(rand(7).cuda()), torch.nn.Parameter((rand(129) + 3).to(dtype).cuda())]
    opt = optim.FusedAdamW(ps, lr=1e-2, master=True)

    def step():
        for p in ps:
            p.grad = (rand(*p.shape) * 0.1 + 0.05).to(p.dtype).cuda()
        opt.step()
    step()
    with torch.no_grad():
        for p in ps:
            p.copy_((rand(*p.shape) - 5).to(p.dtype))
    for p in (ps[0], ps[2]):
        del opt.state[p]["master"]
    for t in (2, 3):
        before = [(f64(opt.state[p].get("master", p)), f64(opt.state[p]["exp_avg"]), f64(opt.state[p]["exp_avg_sq"])) for p in ps]
        step()
        for p, (x, m, v) in zip(ps, before):
            master = opt.state[p]["master"] if p.dtype == dtype else None
            _one_step(x, f64(p.grad), m, v, 1e-2, t, f64(p), None if master is None else f64(master), half if p.dtype == dtype else 0.0)
    mine = torch.full((129,), 7.0, device="cuda")
    opt.state[ps[2]]["master"] = mine
    m, v = f64(opt.state[ps[2]]["exp_avg"]), f64(opt.state[ps[2]]["exp_avg_sq"])
    step()
    _one_step(f64(torch.full((129,), 7.0)), f64(ps[2].grad), m, v, 1e-2, 4, f64(ps[2]), f64(mine), half)


def test_assigned_scales_are_read():
    """The scale of every block doubled by assignment: the step reads moments twice as large, and writes its scales into the assigned tensors."""
    from benerf_amd import optim
    p = torch.nn.Parameter(torch.randn(700, generator=torch.Generator().manual_seed(1)).cuda())
    opt = optim.FusedAdamW([p], lr=1e-2, state_bits=8)
    for _ in range(2):
        p.grad = torch.randn(700, generator=torch.Generator().manual_seed(2)).cuda()
        opt.step()
    st = opt.state[p]
    for name in ("exp_avg_scale", "exp_avg_sq_scale"):
        st[name] = st[name] * 2
    m, u = (optim.decode_moment(st[name], st[name + "_scale"]) for name in ("exp_avg", "exp_avg_sq"))
    before, m, v = f64(p), f64(m), f64(u) ** 2
    held = st["exp_avg_scale"], st["exp_avg_sq_scale"]
    kept = [x.clone() for x in held]
    p.grad = torch.zeros(700, device="cuda")
    opt.step()
    (p2, m2, v2), (dp, _, _, _) = O.step(before, 0 * before, m, v, 1e-2, 3, (0.9, 0.999), 1e-8, 0.01)
    assert (abs(f64(p) - p2) - dp).max() <= 0
    # m shrinks by a tenth and u by 0.05 %: a block's scale stays, or halves where its largest value falls below a power of two
    for x, y, name in zip(held, kept, ("exp_avg_scale", "exp_avg_sq_scale")):
        assert opt.state[p][name] is x and bool(((x == y) | (x == y / 2)).all())


def test_a_32_bit_checkpoint_in_8_bits_moves_no_further():
    """A block whose second moments span 2^36: roots far below the block's largest are lifted, not lost, so the first step in 8 bits is no longer than the
    one in 32 (m and u to nearest, 2^-4 each)."""
    from benerf_amd import optim
    n, lr = 300, 1e-2
    u, m = torch.full((n,), 2.0 ** -18), torch.full((n,), 2.0 ** -18)
    u[0], u[128], u[299], m[0], m[128], m[299] = 1.0, 1.5, 255.0, 0.01, -0.01, 0.01
    moved = []
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
        opt = optim.FusedAdamW([p], lr=lr, weight_decay=0.0, state_bits=bits)
        state = {0: dict(step=torch.tensor(999.0), exp_avg=m.clone(), exp_avg_sq=u.square())}
        opt.load_state_dict(dict(state=state, param_groups=opt.state_dict()["param_groups"]))
        p.grad = torch.zeros_like(p)
        opt.step()
        moved.append(p.detach().abs())
    assert bool((moved[1] <= 1.2 * moved[0]).all()) and bool((moved[0][1:128] > 0.5 * lr).all()) and float(opt.state[p]["step"]) == 1000.0


def _network(seed):
    from benerf_amd.model.nerf import NeRF
    torch.manual_seed(seed)
    return NeRF(D=8, W=256, input_ch=63, input_ch_views=27, output_ch=4, skips=[4], use_viewdirs=True, channels=1).to(DEV)


def _fresh_pack(net):
    """The network's weights packed now; words that packing does not write are those of its own pack."""
    from benerf_amd import kernels as K
    ws, bs = net.param_lists()
    copy = K.PackedMlp([w.detach().clone() for w in ws], [b.detach().clone() for b in bs], net.channels)
    copy.packed.copy_(net.packed().packed)
    copy.pack()
    return copy.packed.view(torch.int32)


def test_renders_after_a_replayed_step_see_its_weights():
    """A captured step changes network weights at every replay, where no generation and no version counter moves: an eager forward and backward
    after each replay run on the weights as they are, and a forward between the two of another changes nothing."""
    from benerf_amd import optim
    net = _network(2)
    params = list(net.parameters())
    opt = optim.FusedAdamW(params, lr=1e-2, capturable=True)
    pts, dirs = torch.rand(33, 2, 3, device=DEV), torch.nn.functional.normalize(torch.randn(33, 3, device=DEV), dim=1)

    def forward(n):
        return n(0, pts, dirs, None)
    for p in params:
        p.grad = torch.randn_like(p)
    opt.step()
    forward(net)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    forward(net)
    seen = []
    for _ in range(3):
        graph.replay()
        out = forward(net)
        torch.cuda.synchronize()
        assert torch.equal(net.packed().packed.view(torch.int32), _fresh_pack(net))
        twin = _network(3)
        twin.load_state_dict(net.state_dict())
        assert torch.equal(out, forward(twin))
        seen.append(out)
        # two forward passes, then the first one's gradients: packed again in between, with the same weights
        other = forward(net)
        grads = torch.autograd.grad(out.sum(), params)
        want = torch.autograd.grad(forward(twin).sum(), list(twin.parameters()))
        assert all(torch.equal(a, b) for a, b in zip(grads, want)) and torch.equal(other, out)
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
    # weights that no captured step writes are packed once
    from benerf_amd import kernels as K
    forward(twin)
    assert not twin.packed().stale() and net.packed().stale()
    assert K.PackedMlp([w.detach().clone() for w in net.packed().weights], net.packed().biases, 1).stale()


def test_a_captured_pack_is_part_of_its_graph():
    """Packed just before the capture or not: a pack inside a capture is recorded, since the weights may be others at a replay."""
    net = _network(4)
    packed = net.packed()
    packed.pack_if_stale()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed.pack_if_stale()
    for k in range(3):
        with torch.no_grad():
            for p in net.parameters():
                p.add_(0.01 * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(packed.packed.view(torch.int32), _fresh_pack(net))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("order", [(0, 5), (5, 0), (0, 0, 700, 0)])
def test_empty_parameters_with_masters(order, bits):
    from benerf_amd import optim
    gen = torch.Generator().manual_seed(7)
    ps = [torch.nn.Parameter((torch.randn(n, generator=gen) + 3).to(torch.bfloat16).cuda()) for n in order]
    start = [f64(p) for p in ps]
    opt = optim.FusedAdamW(ps, lr=1e-2, master=True, max_norm=10.0, state_bits=bits)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    norm = sum(order) ** 0.5
    assert abs(float(opt.grad_norm[0]) - norm) <= 2 * O.HALF * norm
    scale = min(1.0, 10.0 / (norm + 1e-6))
    for p, x in zip(ps, start):
        if x.size:
            (p2, _, _), (dp, _, _, _) = O.step(x, 0 * x + 1, 0 * x, 0 * x, 1e-2, 1, (0.9, 0.999), 1e-8, 0.01, scale)
            master = f64(opt.state[p]["master"])
            assert (abs(master - p2) - dp).max() <= 0 and (abs(f64(p) - master) - 2.0 ** -8 * abs(master)).max() <= 0


PATTERNS = (0x7fc00000, 0xffc00000, 0x7fffffff, 0xffffffff, 0x7f800001, 0xff800001, 0x7fbfffff, 0x7f800000, 0xff800000)


@pytest.mark.parametrize("eps", [1e-8, 1e-15])
@pytest.mark.parametrize("n", [1, 100, 128, 129, 300, 640])
def test_non_finite_gradients_in_8_bits_beside_empty_blocks(n, eps):
    """inf and NaN of every kind in one element of a tensor whose other block of the wavefront is empty, zero or ordinary, over many draws: both codes of
    that element are NaN and stay it, every other element takes the step of the formula, block scales included.  (Bit for bit the others need not be what
    they are without: the root of a wavefront with an empty block is rounded correctly, others to 1 ulp.)"""
    from benerf_amd import kernels as K, optim
    gen = torch.Generator().manual_seed(n)
    clean = torch.randn(n, generator=gen)
    clean[128:256] = 0.0                                               # a block of zeros, if there is one
    for k, word in enumerate(PATTERNS):
        at = (n - 1, 0, n // 2)[k % 3]
        others = np.arange(n) != at
        p = torch.zeros(n, device="cuda")
        moments = optim.zero_moments([p], 8)
        plan = K.AdamWPlan([p], **moments)
        g = clean.clone()
        g.view(torch.int32)[at] = int(np.uint32(word).astype(np.int32))
        g = g.cuda()
        x, m, u = (np.where(others, np.nan_to_num(y), 0.0) for y in (f64(p), np.zeros(n), np.zeros(n)))
        for t in range(1, 9):
            K.adamw_step(plan, [g], 1e-2, t, eps=eps, weight_decay=0.01, seed=k)
            (p2, m2, v2), (dp, dm, dv, du) = O.step(x, np.where(others, f64(clean), 0.0), m, u * u, 1e-2, t, (0.9, 0.999), eps, 0.01)
            assert np.isnan(f64(p)[at]) and np.all(np.abs(f64(p) - p2)[others] <= dp[others]), (hex(word), t)
            got = []
            for name, y, dy, r, keep in (("exp_avg", m2, dm, O.draws(n, 0, t, k)[0], False), ("exp_avg_sq", np.sqrt(v2), du, O.draws(n, 0, t, k)[1], True)):
                code, scale = f64(moments[name][0].float()), f64(moments[name + "_scale"][0])
                assert np.isnan(code[at]), (hex(word), t, name, code[at])
                value = code * np.repeat(scale, 128)[:n]
                low, high = O.coded_range(y, dy, r, keep)
                assert np.all(((low <= np.abs(value)) & (np.abs(value) <= high))[others]), (hex(word), t, name)
                assert np.all((scale >= O.scale_of(np.maximum(np.abs(y) - dy, 0))) & (scale <= O.scale_of(np.abs(y) + dy))), (hex(word), t, name)
                got.append(value)
            x, m, u = (np.where(others, y, 0.0) for y in (f64(p), *got))


@pytest.mark.parametrize("every", [1, 4])
def test_steps_skipped_by_the_norm_are_reported(every):
    """A norm that is not finite step after step: the networks stay, and step() raises from the copies that it keeps of the counters, without a
    synchronisation of its own; a single skipped step passes; steps that the range guard skips are not counted here; check_range() sees both."""
    from benerf_amd import _lib, engine, kernels as K
    args, cam, HW, accu, img = _setting(benerf_optimizer="adamw", benerf_max_grad_norm=1.0)
    _, g = _graph(args, seed=3)
    step = engine.TrainStep(g, args, cam, cam, torch.device(DEV), seed=21)
    step.GUARD_POST_EVERY = every
    real = K.grad_norm

    def poisoned(grads, *a, **kw):
        step.flat_g[5] = float("nan")
        return real(grads, *a, **kw)

    def run(n, bad):
        K.grad_norm = poisoned if bad else real
        try:
            for _ in range(n):
                _run(step, HW, accu, img, step.global_step, step.global_step + 1)
                torch.cuda.synchronize()
        finally:
            K.grad_norm = real
    run(3, False)
    step.check_range()
    run(2, True)
    run(2 * every, False)                     # a short run of skips is no error while training
    with pytest.raises(_lib.BenerfRangeError, match="norm"):
        step.check_range()
    step.check_range()                        # told once
    before = step.flat_p[:2 * step.n_net].clone()
    knots = step.knots.clone()
    at = step.global_step
    with pytest.raises(_lib.BenerfRangeError, match="norm"):
        run(3 * max(every, 3), True)
    assert step.global_step - at <= 2 * every + 3 and torch.equal(step.flat_p[:2 * step.n_net], before)
    # the trajectory, whose gradients were finite, went on; nothing of it is gated by the networks' norm
    assert bool(step.flat_p[2 * step.n_net:].isfinite().all()) and not torch.equal(step.knots, knots)
    run(2 * every, False)                     # told once, and training goes on
    assert not torch.equal(step.flat_p[:2 * step.n_net], before)
    # the guard's own skips are its own: [SKIP] set for every step by a poisoned verdict
    step.check_range()
    total = float(step.net_norm[3])
    gate = step.guard.gate

    def closed(flag=None, phase=1):
        step.guard.words[_lib.ST_ACT] = 0x7f800000
        gate(flag, phase)
    step.guard.gate = closed
    with pytest.raises(_lib.BenerfRangeError, match="f16 range"):
        run(3 * max(every, 3), False)
    step.guard.gate = gate
    assert float(step.net_norm[3]) >= total + 3
    with pytest.raises(_lib.BenerfRangeError, match="f16 range"):
        step.check_range()
    step.check_range()
    run(2 * every, False)


def test_tables_of_captured_plans_can_be_released():
    """Captures with plans that are let go: their tables stay, and go when they are released; a graph whose plan lives replays on."""
    import gc
    from benerf_amd import _lib, kernels as K, optim

    def capture():
        p, g = [torch.ones(100000, device="cuda")], [torch.ones(100000, device="cuda")]
        plan = K.AdamWPlan(p, **optim.zero_moments(p, 32))
        grads, step = K.GradList(g, plan), torch.zeros((), device="cuda")
        K.grad_norm(grads, counters=[step])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.grad_norm(grads, counters=[step])
            K.adamw_step(plan, grads, 1e-2, step, weight_decay=0.0)
        return p, plan, grads, step, graph
    K.release_captured()
    kept = capture()
    assert len(K._captured) == 1
    for _ in range(4):
        capture()
    gc.collect()
    tables = 80 * 196 * 4                       # 196 pieces of 512 elements each
    held = torch.cuda.memory_allocated()
    assert len(K._captured) == 5
    K.release_captured()
    gc.collect()
    assert not K._captured and held - torch.cuda.memory_allocated() >= tables
    filled = [torch.full((16 << 10,), 255, dtype=torch.uint8, device="cuda") for _ in range(64)]
    p, plan, grads, step, graph = kept
    for t in (2, 3, 4):
        graph.replay()
        torch.cuda.synchronize()
        # gradients of ones: m / (1 - b1^t) and v / (1 - b2^t) are 1 after steps 1 .. t, and the first here is t = 2 on moments of zero
        assert float(step) == t and bool((p[0] == p[0][0]).all())
    assert 1.0 - 3 * 1e-2 * 1.1 <= float(p[0][0]) < 1.0 and len(filled) == 64
    refused = []
    side = torch.cuda.CUDAGraph()
    with torch.cuda.graph(side):
        torch.zeros(1, device="cuda")
        try:
            K.release_captured()
        except _lib.BenerfHipError as e:
            refused.append(str(e))
    assert refused


@pytest.mark.parametrize("precision", ["split", "split_f16bwd", "f32"])
def test_a_network_trained_inside_a_graph(precision):
    """Forward, backward and step of a network on its points in one graph, replayed several times beside eager work on another network: every replay's loss
    and weights are those of an eager twin."""
    from benerf_amd import kernels as K, optim
    K.set_mlp_precision(precision)
    try:
        gen = torch.Generator().manual_seed(6)
        batches = [(torch.rand(40, 3, 3, generator=gen).to(DEV), torch.nn.functional.normalize(torch.randn(40, 3, generator=gen), dim=1).to(DEV)) for _ in range(8)]

        def build():
            net = _network(5)
            return net, optim.FusedAdamW(net.parameters(), lr=1e-3, capturable=True, max_norm=1.0)

        def once(net, opt, pts, dirs):
            opt.zero_grad(set_to_none=True)
            loss = (net(0, pts, dirs, None) ** 2).mean()
            loss.backward()
            opt.step()
            return loss.detach()
        (na, a), (nb, b) = build(), build()
        other = _network(7)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for k in range(2):
                once(na, a, *batches[k])
                once(nb, b, *batches[k])
        torch.cuda.current_stream().wait_stream(side)
        held = [x.clone() for x in batches[0]]
        graph = torch.cuda.CUDAGraph()
        a.zero_grad(set_to_none=True)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            la = once(na, a, *held)
        for k in range(2, 8):
            for x, y in zip(held, batches[k]):
                x.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            lb = once(nb, b, *batches[k])
            assert float(la) == float(lb), k
            for p, q in zip(na.parameters(), nb.parameters()):
                assert torch.equal(p, q), k
            with torch.no_grad():
                out = other(0, *batches[k - 1], None)          # an inference launch, and a render of the trained network
                assert torch.equal(na(0, *batches[k - 1], None), nb(0, *batches[k - 1], None)) and bool(out.isfinite().all())
            torch.cuda.synchronize()
        assert float(a.state[next(na.parameters())]["step"]) == 8.0 and float(a.grad_norm[3]) == 0.0
    finally:
        K.set_mlp_precision("split")


def test_a_captured_inference_launch():
    """An inference launch of a network, captured and replayed over changing weights and points: its own overflow word starts from zero every time."""
    net = _network(8)
    twin = _network(8)
    gen = torch.Generator().manual_seed(9)
    batches = [(torch.rand(40, 3, 3, generator=gen).to(DEV), torch.nn.functional.normalize(torch.randn(40, 3, generator=gen), dim=1).to(DEV)) for _ in range(6)]
    held = [x.clone() for x in batches[0]]
    with torch.no_grad():
        net(0, *held, None)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = net(0, *held, None)
        for k in range(6):
            # every second time the first layer overflows float16, so that the launch falls back to float32; the next one must not
            with torch.no_grad():
                for n in (net, twin):
                    for li, layer in enumerate(n.pts_linears):
                        layer.weight.mul_((300.0 if li == 0 else 3.0) if k % 2 else (1 / 300.0 if li == 0 else 1 / 3.0) if k else 1.0)
            for x, y in zip(held, batches[k]):
                x.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, twin(0, *batches[k], None)), k
            torch.cuda.synchronize()
