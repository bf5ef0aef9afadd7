"""CPU: what becomes of optimiser state outside the kernels - checkpoints of one form read by the other - with the real host code on host tensors."""
from types import SimpleNamespace

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
        self.crf_groups, self.global_step = [], 0
        self.guard = SimpleNamespace(words=torch.zeros(16, dtype=torch.int32))
        packed = SimpleNamespace(packed=SimpleNamespace(pack=lambda: None))
        self.net_c = self.net_f = packed
        for name in ("_lr", "_flat_slice", "_network_places", "_trained_optimizers", "import_optimizer_state"):
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
