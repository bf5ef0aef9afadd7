"""GPU: the framework's own paths with AdamW for the networks (args.benerf_optimizer): Model.setup_optimizer, the fused TrainStep,
checkpoints between them."""
import copy

import numpy as np
import pytest
import torch

from test_api_gpu import DEV, _graph

pytestmark = pytest.mark.gpu


def _setting(**over):
    from benerf_amd import engine, workloads as WL
    wl = dict(WL.WORKLOADS["C1"], S=16, Ni=16, Re=32, Rr=4, n=5)
    args = WL.make_args(wl, **over)
    cam = WL.CAMERAS[wl["cam"]]
    cam_o = engine.Camera(cam["H"], cam["W"], cam["fx"], cam["fy"], cam["cx"], cam["cy"])
    rng = np.random.default_rng(5)
    HW = cam["H"] * cam["W"]
    accu = torch.from_numpy(rng.integers(-3, 4, HW).astype(np.float32)).to(DEV)
    img = torch.from_numpy(rng.random((HW, 1)).astype(np.float32)).to(DEV)
    return args, cam_o, HW, accu, img


def _run(step, HW, accu, img, n0, n1):
    from benerf_amd import kernels as K
    ts_e, ts_r = torch.tensor([0.2, 0.3], device=DEV), torch.tensor([0.0, 1.0], device=DEV)
    for it in range(n0, n1):
        step.step(ts_e, ts_r, K.sample_pixels(HW, 32, 9, 2 * it, torch.device(DEV)), K.sample_pixels(HW, 4, 9, 2 * it + 1, torch.device(DEV)), accu, img)


def test_setup_optimizer_and_refusals():
    from benerf_amd import engine, optim
    args, cam, *_ = _setting(benerf_optimizer="adamw8", benerf_max_grad_norm=0.5, benerf_weight_decay=0.02)
    model, g = _graph(args)
    nerf, pose, trans, rgb, evt = model.setup_optimizer(args)
    assert type(nerf) is optim.FusedAdamW and nerf.state_bits == 8 and nerf.max_norm == 0.5 and nerf.param_groups[0]["weight_decay"] == 0.02
    assert all(type(o) is optim.FlatAdam for o in (pose, trans, rgb, evt))
    model, g = _graph(_setting()[0])
    assert type(model.setup_optimizer(_setting()[0])[0]) is optim.FlatAdam
    for over in (dict(benerf_optimizer="sgd"), dict(benerf_max_grad_norm=1.0), dict(benerf_weight_decay=0.1)):
        bad = _setting(**over)[0]
        with pytest.raises(ValueError):
            model.setup_optimizer(bad)
        with pytest.raises(ValueError):
            engine.TrainStep(g, bad, cam, cam, torch.device(DEV))


def test_train_step_without_decay_is_adam():
    """AdamW with no decay is Adam: the fused step with either optimiser walks the same way, to rounding."""
    from benerf_amd import engine
    got = []
    for over in (dict(), dict(benerf_optimizer="adamw", benerf_weight_decay=0.0)):
        args, cam, HW, accu, img = _setting(**over)
        _, g = _graph(args, seed=3)
        step = engine.TrainStep(g, args, cam, cam, torch.device(DEV), seed=21)
        start = step.flat_p.clone()
        _run(step, HW, accu, img, 0, 1)
        got.append((start, step.flat_p.clone(), step.flat_g.clone(), step.flat_m.clone(), step.flat_v.clone()))
    (s0, p0, g0, m0, v0), (s1, p1, g1, m1, v1) = got
    assert torch.equal(s0, s1) and torch.equal(g0, g1)
    assert torch.equal(m0, m1) and torch.equal(v0, v1)
    # one step of at most lr: 16 roundings of it, 3 of the weight
    assert float(((p0 - p1).abs() - 2.0 ** -24 * (3 * p0.abs() + 16 * 5e-4)).max()) <= 0


@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_train_step_clips_and_resumes(tmp_path, kind):
    """Clipped steps; a checkpoint through Model.setup_optimizer's objects into another TrainStep goes on with the same bits."""
    from benerf_amd import checkpoint as CK, engine
    args, cam, HW, accu, img = _setting(benerf_optimizer=kind, benerf_max_grad_norm=0.01)
    model_a, g_a = _graph(args, seed=3)
    a = engine.TrainStep(g_a, args, cam, cam, torch.device(DEV), seed=21)
    _run(a, HW, accu, img, 0, 3)
    n = 2 * a.n_net
    norm = float(a.flat_g[:n].double().norm())
    assert abs(float(a.net_norm[0]) - norm) <= 1e-6 * norm and norm > 0.01 and abs(float(a.net_norm[1]) - 0.01 / norm) <= 1e-6
    assert float(a.net_steps) == 3.0 and a.flat_m.numel() == a.flat_p.numel() - (n if kind == "adamw8" else 0)
    optims = model_a.setup_optimizer(args)
    a.export_optimizer_state(optims)
    path = str(tmp_path / "ck.tar")
    CK.save(path, g_a, optims, a.global_step)
    model_b, g_b = _graph(args, seed=8)
    ob = model_b.setup_optimizer(args)
    b = engine.TrainStep(g_b, args, cam, cam, torch.device(DEV), seed=21)
    b.import_optimizer_state(ob, CK.load(path, g_b, ob))
    for s in (a, b):
        _run(s, HW, accu, img, 3, 5)
    assert torch.equal(a.flat_p, b.flat_p) and torch.equal(a.flat_m, b.flat_m) and float(b.net_steps) == 5.0
    for name in a.net_moments:
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.net_moments[name], b.net_moments[name]))


def test_train_step_skips_what_is_not_finite():
    """A NaN in one gradient between the backward pass and the optimiser: the range guard cannot have seen it, the norm does."""
    from benerf_amd import engine, kernels as K
    args, cam, HW, accu, img = _setting(benerf_optimizer="adamw8", benerf_max_grad_norm=1.0)
    _, g = _graph(args, seed=3)
    step = engine.TrainStep(g, args, cam, cam, torch.device(DEV), seed=21)
    _run(step, HW, accu, img, 0, 1)
    real = K.grad_norm

    def poisoned(grads, *a, **kw):
        step.flat_g[5] = float("nan")
        return real(grads, *a, **kw)
    before = step.flat_p[:2 * step.n_net].clone()
    K.grad_norm = poisoned
    try:
        _run(step, HW, accu, img, 1, 2)
    finally:
        K.grad_norm = real
    assert torch.equal(step.flat_p[:2 * step.n_net], before) and float(step.net_steps) == 1.0 and float(step.net_norm[3]) == 1.0
    _run(step, HW, accu, img, 2, 3)
    assert not torch.equal(step.flat_p[:2 * step.n_net], before) and float(step.net_steps) == 2.0


@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_reference_shaped_iterations(kind):
    """render, loss, backward, the optimisers of Model.setup_optimizer - the networks' weights against torch's AdamW on the same
    gradients; renders see the new weights."""
    args, cam, HW, accu, img = _setting(benerf_optimizer=kind, benerf_max_grad_norm=0.05)
    model, g = _graph(args, seed=3)
    nerf = model.setup_optimizer(args)[0]
    params = list(nerf.param_groups[0]["params"])
    twins = [torch.nn.Parameter(p.detach().double().cpu()) for p in params]
    ref = torch.optim.AdamW(twins, lr=args.lrate, weight_decay=0.01)
    Km = np.array([[548.409, 0, 384.0], [0, 548.409, 240.0], [0, 0, 1]])
    idx = torch.arange(0, 64, device=DEV)
    seen = []
    for it in range(3):
        torch.manual_seed(it)
        nerf.zero_grad()
        poses = g.get_pose_rgb(args, torch.tensor([0.0, 1.0]))
        ret = g.render(it, poses, idx, 480, 768, Km, args, enable_crf=False, sensor_type=None, remap=None, training=True)
        loss = ((ret["rgb_map"] - 0.3) ** 2).mean() + ((ret["rgb0"] - 0.3) ** 2).mean()
        loss.backward()
        for p, t in zip(params, twins):
            t.grad = p.grad.double().cpu()
        torch.nn.utils.clip_grad_norm_(twins, 0.05)
        nerf.step()
        ref.step()
        seen.append(float(loss))
    # moments in 32 bits: 4 roundings of the weight a step and 200 of the rate; the first update in 8 bits is that of 32 (moments of zero)
    room = 3 * (4 * 2.0 ** -24 + 200 * 2.0 ** -24 * args.lrate)
    worst = max(float((p.detach().double().cpu() - t.detach()).abs().max()) for p, t in zip(params, twins))
    assert worst <= (room if kind == "adamw" else 2 * args.lrate), worst
    assert len(set(seen)) == 3 and all(np.isfinite(seen))


@pytest.mark.parametrize("decay", [0.01, 0.0])
def test_eight_bit_checkpoint_into_flat_adam(decay):
    """FlatAdam reads the 8-bit form too: as the values, not the codes.  It goes on refusing decay, a loaded one as well."""
    from benerf_amd import optim
    p = torch.nn.Parameter(torch.zeros(300, device=DEV))
    a = optim.FusedAdamW([p], state_bits=8, seed=1, weight_decay=decay)
    for it in range(2):
        p.grad = torch.randn(300, device=DEV) * 1e-3
        a.step()
    want = optim.decode_moment(a.state[p]["exp_avg"], a.state[p]["exp_avg_scale"])
    q = torch.nn.Parameter(p.detach().clone())
    b = optim.FlatAdam([q], lr=1e-3)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    q.grad = torch.zeros(300, device=DEV)
    if decay:
        with pytest.raises(NotImplementedError):
            b.step()
        return
    b.step()
    assert torch.allclose(b.state[q]["exp_avg"], want * 0.9, rtol=1e-6, atol=0) and float(b.state[q]["step"]) == 3.0
