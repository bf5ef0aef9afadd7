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
