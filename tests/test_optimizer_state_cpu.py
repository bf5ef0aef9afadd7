"""CPU: what becomes of optimiser state outside the kernels - checkpoints of one form read by the other - with the real host code on host tensors."""
import ctypes
import os
from types import SimpleNamespace

import pytest
import torch

LR = 5e-4


def _eight_bit(n, seed):
    """A parameter's state as FusedAdamW(state_bits=8) saves it, and the float32 moments that it stands for."""
    from benerf_amd import optim
    gen = torch.Generator().manual_seed(seed)
    m, u = torch.randn(n, generator=gen) * 1e-3, torch.randn(n, generator=gen).abs() * 1e-4 + 1e-6
    st = {"step": torch.tensor(7.0)}
    st["exp_avg"], st["exp_avg_scale"] = optim.encode_moment(m)
    st["exp_avg_sq"], st["exp_avg_sq_scale"] = optim.encode_moment(u)
    return st, optim.decode_moment(st["exp_avg"], st["exp_avg_scale"]), optim.decode_moment(st["exp_avg_sq"], st["exp_avg_sq_scale"]).square()


class _Step:
    """A TrainStep's flat buffers without a GPU, two network parameters of 300 and 5 values and one of the trajectory; net_bits as there."""

    def __init__(self, net_bits):
        from benerf_amd import engine, optim
        n = 305
        self.flat_p, self.off_moments, self.net_bits = torch.zeros(n + 24), n if net_bits == 8 else 0, net_bits
        self.flat_m, self.flat_v = torch.full((n + 24 - self.off_moments,), 9.0), torch.full((n + 24 - self.off_moments,), 9.0)
        nets = [self.flat_p[:300], self.flat_p[300:305]]
        self.params = [torch.nn.Parameter(x) for x in nets + [self.flat_p[305:]]]
        self.net_plan, self.net_steps = None, torch.zeros(())
        if net_bits is not None:
            self.net_plan = SimpleNamespace(params=nets)
            self.net_moments = optim.zero_moments(nets, 8) if net_bits == 8 else \
                {"exp_avg": [self.flat_m[:300], self.flat_m[300:305]], "exp_avg_sq": [self.flat_v[:300], self.flat_v[300:305]]}
        self.cfg = SimpleNamespace(lrate=LR, decay_rate=0.1, pose_lrate=LR, decay_rate_pose=0.1, transform_lrate=LR, decay_rate_transform=0.1, lrate_decay=10)
        self.crf_groups, self.global_step, self.max_grad_norm = [], 0, None
        self.guard = SimpleNamespace(words=torch.zeros(16, dtype=torch.int32))
        packed = SimpleNamespace(packed=SimpleNamespace(pack=lambda: None))
        self.net_c = self.net_f = packed
        for name in ("_lr", "_flat_slice", "_network_places", "_trained_optimizers", "_norm_from_here", "import_optimizer_state"):
            setattr(self, name, getattr(engine.TrainStep, name).__get__(self))

    def moments(self, k):
        a, b = ((0, 300), (300, 305))[k]
        if self.net_bits is None:
            return self.flat_m[a:b], self.flat_v[a:b]
        from benerf_amd import optim
        held = optim.convert_moments({name: ts[k] for name, ts in self.net_moments.items()}, 32)
        return held["exp_avg"], held["exp_avg_sq"]


def test_eight_bit_checkpoint_into_a_train_step():
    """The moments that an 8-bit checkpoint stands for arrive whichever optimiser the networks have: Adam's flat range, AdamW in 32 bits, AdamW in 8
    bits; from the optimiser object in either form (FlatAdam's load turns the codes into float32 numbers and leaves them codes)."""
    for net_bits in (None, 32, 8):
        for as_float in (False, True):
            step = _Step(net_bits)
            saved = [_eight_bit(n, seed) for n, seed in ((300, 1), (5, 2))]
            nerf = SimpleNamespace(param_groups=[dict(params=step.params[:2])], state={})
            for p, (st, _, _) in zip(step.params, saved):
                nerf.state[p] = {k: v.float() if as_float else v for k, v in st.items()}
            pose = SimpleNamespace(param_groups=[dict(params=step.params[2:])],
                                   state={step.params[2]: dict(step=torch.tensor(7.0), exp_avg=torch.full((24,), 0.5), exp_avg_sq=torch.full((24,), 0.25))})
            step.import_optimizer_state((nerf, pose, SimpleNamespace(param_groups=[], state={})), 9)
            for k, (_, m, v) in enumerate(saved):
                got_m, got_v = step.moments(k)
                assert torch.equal(got_m, m) and torch.equal(got_v, v), (net_bits, as_float, k)
            assert torch.equal(step.flat_m[305 - step.off_moments:], torch.full((24,), 0.5)) and torch.equal(step.flat_v[305 - step.off_moments:], torch.full((24,), 0.25))
            assert step.global_step == 9 and int(step.guard.words[12]) == 2
            assert net_bits is None or float(step.net_steps) == 7.0


class _Plan:
    """Stands for kernels.AdamWPlan on the host: remembers what it was made of."""
    made = []

    def __init__(self, params, exp_avg, exp_avg_sq, exp_avg_scale=None, exp_avg_sq_scale=None, master=None):
        self.params, self.numels, self.device, self.parts = params, [p.numel() for p in params], SimpleNamespace(index=-1), []
        self.state_bits, self.master = 32 if exp_avg_scale is None else 8, master
        self.held = dict(exp_avg=exp_avg, exp_avg_sq=exp_avg_sq, exp_avg_scale=exp_avg_scale, exp_avg_sq_scale=exp_avg_sq_scale, master=master)
        _Plan.made.append(self)


@pytest.fixture
def plans(monkeypatch):
    """FusedAdamW without a GPU: plans are _Plan, a step marks what it would write (masters + 1, rounded into their parameters)."""
    from benerf_amd import kernels as K
    _Plan.made = []

    def step(plan, grads, *a, **kw):
        for k, p in enumerate(plan.params):
            x = plan.held["master"][k] if plan.held["master"] else None
            (p if x is None else x).add_(1.0)
            if x is not None:
                p.copy_(x)
    monkeypatch.setattr(K, "AdamWPlan", _Plan)
    monkeypatch.setattr(K.GradList, "of_checked", classmethod(lambda cls, grads, plan: grads))
    monkeypatch.setattr(K, "adamw_step", step)
    return _Plan.made


def _steps(opt, params, n=1):
    for _ in range(n):
        for p in params:
            p.grad = torch.ones_like(p)
        opt.step()


def test_dropped_and_assigned_masters_are_followed(plans):
    """Weights loaded in place after a step and their masters dropped: the next step starts from the loaded weights and there are masters again; an
    assigned master is the one that is read and written; without either the plan stays."""
    from benerf_amd import optim
    params = [torch.nn.Parameter(torch.zeros(5, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(4, dtype=torch.float16))]
    opt = optim.FusedAdamW(params, master=True)
    _steps(opt, params, 3)
    assert len(plans) == 1 and all(torch.equal(p, torch.full_like(p, 3.0)) for p in params) and "master" not in opt.state[params[1]]
    with torch.no_grad():
        for p in params:
            p.fill_(8.0)
    for p in (params[0], params[2]):
        del opt.state[p]["master"]
    _steps(opt, params)
    assert all(torch.equal(p, torch.full_like(p, 9.0)) for p in params), params
    assert all(torch.equal(opt.state[p]["master"], torch.full(p.shape, 9.0)) for p in (params[0], params[2])) and len(plans) == 2
    assert float(opt.state[params[0]]["step"]) == 4.0
    mine = torch.full((4,), 20.0)
    opt.state[params[2]]["master"] = mine
    _steps(opt, params, 2)
    assert torch.equal(mine, torch.full((4,), 22.0)) and torch.equal(params[2], torch.full_like(params[2], 22.0)) and len(plans) == 3
    assert "master" in opt.state_dict()["state"][0]


def test_dropped_and_assigned_moments_are_followed(plans):
    """Codes, scales and counters that are assigned are the ones of the next step; moments that are dropped start at zero, codes without their
    scales are refused."""
    from benerf_amd import optim
    params = [torch.nn.Parameter(torch.zeros(300)), torch.nn.Parameter(torch.zeros(5))]
    opt = optim.FusedAdamW(params, state_bits=8)
    _steps(opt, params, 2)
    assert len(plans) == 1
    for count, name in enumerate(("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step"), 2):
        opt.state[params[0]][name] = opt.state[params[0]][name].clone()
        _steps(opt, params, 2)
        assert len(plans) == count, name
        if name != "step":
            assert plans[-1].held[name][0] is opt.state[params[0]][name]
    st = opt.state[params[1]]
    for name in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"):
        del st[name]
    _steps(opt, params)
    assert plans[-1].held["exp_avg_scale"][1] is st["exp_avg_scale"] and not st["exp_avg"].float().any() and float(st["step"]) == 13.0
    del st["exp_avg_sq_scale"], st["exp_avg_scale"]
    for p in params:
        p.grad = torch.ones_like(p)
    with pytest.raises(ValueError):
        opt.step()


def test_encoded_roots_above_zero_stay_above_zero():
    """Of the second moment's root no value above 0 may become 0: with m on a scale of its own the next update would be divided by eps alone.  A
    32-bit checkpoint in 8 bits takes the step that it takes in 32."""
    from benerf_amd import optim
    n = 300
    u, m = torch.full((n,), 2.0 ** -18), torch.full((n,), 2.0 ** -18)
    u[0], u[128], u[299], m[0], m[128], m[299] = 1.0, 1.5, 255.0, 0.01, -0.01, 0.01
    u[5], m[5] = 0.0, 0.0
    held = optim.convert_moments(dict(exp_avg=m, exp_avg_sq=u.square()), 8)
    root = optim.decode_moment(held["exp_avg_sq"], held["exp_avg_sq_scale"])
    least = 2.0 ** -9 * held["exp_avg_sq_scale"].repeat_interleave(128)[:n]
    assert bool((root[u > 0] >= least[u > 0]).all()) and root[5] == 0
    # values that nearest does not take to 0 are as they were, and moments with a sign may become 0
    plain = optim.decode_moment(*optim.encode_moment(u))
    assert torch.equal(root[plain > 0], plain[plain > 0]) and bool((plain[1:5] == 0).all())
    assert bool((optim.decode_moment(*optim.encode_moment(torch.tensor([1.0, 2.0 ** -18, -2.0 ** -18])))[1:] == 0).all())
    # the next step without a gradient, t = 1000: its size against the same in 32 bits
    m8 = optim.decode_moment(held["exp_avg"], held["exp_avg_scale"])
    bc2 = (1 - 0.999 ** 1000) ** 0.5
    move8, move32 = (0.9 * x / (0.999 ** 0.5 * y / bc2 + 1e-8) for x, y in ((m8, root), (m, u)))
    # a root is lifted, not lowered, here; m and u are powers of two or rounded to nearest by 2^-4 each
    assert bool((move8.abs() <= 1.2 * move32.abs()).all())
    # not finite: the elements of their own; an empty tensor
    bad = optim.convert_moments(dict(exp_avg=torch.zeros(3), exp_avg_sq=torch.tensor([1.0, float("inf"), float("nan")])), 8)
    assert bad["exp_avg_sq"].float()[1:].isnan().all() and optim.decode_moment(bad["exp_avg_sq"], bad["exp_avg_sq_scale"])[0] == 1.0
    assert optim.convert_moments(dict(exp_avg=torch.zeros(0), exp_avg_sq=torch.zeros(0)), 8)["exp_avg_sq"].shape == (0,)


def test_plans_whose_first_tensor_is_empty():
    """An empty tensor has no memory, so neither masters nor anything else is read off it: wherever it stands, a list with masters is laid out, and
    the others must all have theirs or none."""
    from benerf_amd import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    lib = _lib.load()

    def fill(*rows, kind=1):
        table = (_lib.AdamwTensor * len(rows))(*[_lib.AdamwTensor(**r) for r in rows])
        size = lib.benerf_adamw_plan_bytes(table, len(rows))
        buf = ctypes.create_string_buffer(size)
        return lib.benerf_adamw_plan_fill(table, len(rows), kind, 32, buf, size), bytes(buf)[:48]
    none = dict(n=0)
    full = dict(param=0x1000, exp_avg=0x2000, exp_avg_sq=0x3000, n=5)
    kept = dict(full, master=0x4000)
    heads = [fill(*rows) for rows in ((kept, none), (none, kept), (none, none, kept, none), (kept, kept))]
    assert [rc for rc, _ in heads] == [0, 0, 0, 0]
    assert heads[0][1] == heads[1][1]                                   # type, bits, masters and shape are those of the same list in another order
    assert fill(none, full)[0] == 0 and fill(none)[0] == 0 and fill(none, none)[0] == 0
    for bad in ((none, kept, full), (none, full, kept), (full, none, kept)):
        assert fill(*bad)[0] == -1 and b"master copies" in lib.benerf_last_error()
    assert fill(none, kept, kind=0)[0] == -1 and b"its own master" in lib.benerf_last_error()
    # past the caches from 320 MB on: 13 M bfloat16 with masters (2 + 2 + 8 + 4 bytes) and 30 M are on either side, an empty first tensor or not
    for n in (13 << 20, 30 << 20):
        assert fill(dict(kept, n=n), none)[1] == fill(none, dict(kept, n=n))[1]


def test_what_a_caller_keeps_in_the_state_is_left_alone(plans):
    """Entries of the caller's own come and go without a new plan; together with a replaced or dropped tensor they hide nothing."""
    from benerf_amd import optim
    params = [torch.nn.Parameter(torch.zeros(5, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(3))]
    opt = optim.FusedAdamW(params, master=True)
    _steps(opt, params)
    for p in params:
        for value in (1, 2):
            opt.state[p]["mine"] = value
            _steps(opt, params)
        del opt.state[p]["mine"]
        _steps(opt, params)
    assert len(plans) == 1 and float(opt.state[params[0]]["step"]) == 7.0
    del opt.state[params[0]]["master"]
    opt.state[params[0]]["mine"] = 1            # as many entries as before
    _steps(opt, params)
    assert len(plans) == 2 and "master" in opt.state[params[0]]
    last = opt.state[params[1]]
    del last["step"]                            # the last entry of all, or not
    _steps(opt, params)
    assert len(plans) == 3 and float(last["step"]) == 1.0 and float(opt.state[params[0]]["step"]) == 9.0
