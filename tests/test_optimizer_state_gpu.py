"""GPU: optimiser state between forms and owners - checkpoints of one networks' optimiser resumed with another."""
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
    f64 = lambda t: t.detach().double().cpu().numpy().reshape(-1)      # noqa: E731
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
    f64 = lambda t: t.detach().double().cpu().numpy().reshape(-1)      # noqa: E731
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
