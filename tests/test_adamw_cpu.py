"""CPU: what the optimiser operators over lists (K9) refuse, their host-side plan, the 8-bit codec, and the oracle's own generator."""
import ctypes
import os

import numpy as np
import pytest
import torch

import adamw_oracle as O


@pytest.fixture(scope="module")
def lib():
    from benerf_amd import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


def _rows(*ns, **kw):
    from benerf_amd import _lib
    return (_lib.AdamwTensor * len(ns))(*[_lib.AdamwTensor(**dict(dict(param=0x1000, exp_avg=0x2000, exp_avg_sq=0x3000, n=n, first_block=0), **kw)) for n in ns])


def _fill(lib, rows, kind=0, bits=32, short=0):
    size = lib.benerf_adamw_plan_bytes(rows, len(rows))
    buf = ctypes.create_string_buffer(max(size, 1))
    return lib.benerf_adamw_plan_fill(rows, len(rows), kind, bits, buf, size - short), buf


def test_plan_sizes(lib):
    # header 64, 16 bytes a tensor, 80 bytes a chunk of 512 elements
    size = lambda *ns: lib.benerf_adamw_plan_bytes(_rows(*ns), len(ns))      # noqa: E731
    assert size(1) == 64 + 16 + 80 and size(512, 513, 0) == 64 + 3 * 16 + 80 * 3 and size(1 << 30) == 64 + 16 + (80 << 21)
    # fewer than 2^24 chunks in all
    assert size((1 << 33) - 512) == 64 + 16 + 80 * ((1 << 24) - 1) and size((1 << 33) - 511) == 0 and size(1 << 32, 1 << 32) == 0 and size(*[1 << 40] * 64) == 0
    assert size(-1) == 0 and size(1 << 41) == 0 and lib.benerf_adamw_plan_bytes(None, 1) == 0


def test_plan_refusals(lib):
    from benerf_amd import _lib
    assert _fill(lib, _rows(5))[0] == 0
    for bad, kw in ((_rows(5), dict(kind=3)), (_rows(5), dict(bits=16)), (_rows(5, param=None), {}), (_rows(5, exp_avg=None), {}), (_rows(5), dict(bits=8)),
                    (_rows(5, master=0x4000), {}), (_rows(5, param=0x1002), {}), (_rows(5, exp_avg_sq=0x3002), {}), (_rows(5, first_block=-1), {})):
        rc, _ = _fill(lib, bad, **kw)
        assert rc == -1 and b"adamw_plan_fill" in lib.benerf_last_error()
    assert _fill(lib, _rows(5), short=1)[0] == -2
    mixed = (_lib.AdamwTensor * 2)(_lib.AdamwTensor(param=2, exp_avg=4, exp_avg_sq=4, master=4, n=1), _lib.AdamwTensor(param=2, exp_avg=4, exp_avg_sq=4, n=1))
    assert _fill(lib, mixed, kind=1)[0] == -1
    assert _fill(lib, _rows(0, param=None, exp_avg=None, exp_avg_sq=None))[0] == 0          # an empty tensor has no memory


def test_step_and_norm_refusals(lib):
    from benerf_amd import _lib
    _, plan = _fill(lib, _rows(5))
    _, only = _fill(lib, _rows(5), bits=0)
    g = (ctypes.c_void_p * 1)(0x5000)
    odd = (ctypes.c_void_p * 1)(0x5001)

    def cfg(**kw):
        return ctypes.byref(_lib.AdamwCfg(**dict(dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, step=1), **kw)))
    step = lib.benerf_adamw_step
    for args in ((None, plan, g, 0, cfg()), (plan, None, g, 0, cfg()), (plan, plan, None, 0, cfg()), (plan, plan, g, 3, cfg()), (plan, plan, g, 0, None),
                 (only, only, g, 0, cfg()), (plan, plan, odd, 0, cfg()), (plan, plan, g, 0, cfg(step=0)), (plan, plan, g, 0, cfg(beta1=1.0)),
                 (plan, plan, g, 0, cfg(beta2=-0.1)), (plan, plan, g, 0, cfg(eps=-1.0)), (plan, plan, g, 0, cfg(weight_decay=-1.0)),
                 (ctypes.create_string_buffer(200), plan, g, 0, cfg())):
        assert step(*args, None, None, None) == -1 and b"adamw_step" in lib.benerf_last_error()
    none = (ctypes.c_void_p * 1)()
    assert step(plan, plan, none, 0, cfg(), None, None, None) == 0           # no gradient at all: nothing to launch
    assert lib.benerf_adamw_count(None, None, None, None) == -1
    assert lib.benerf_grad_norm_partials(plan) == 1 and lib.benerf_grad_norm_partials(None) == 0
    keep = []

    def norm(g=g, kind=0, host=plan, dev=0x8000, room=1, most=1.0, words=0x7000, partials=0x6000, counters=None, n=0, rows=1):
        row = (_lib.GradListRow * 1)((None if host is None else ctypes.addressof(host), dev, ctypes.addressof(g) if g is not None else None, kind))
        keep.append(row)
        return lib.benerf_grad_norm(row, rows, partials, room, most, 1.0, words, 0, None, counters, n, None)
    for kw in (dict(g=odd), dict(g=None), dict(kind=3), dict(host=None), dict(dev=None), dict(most=0.0), dict(most=float("nan")), dict(words=None), dict(partials=None),
               dict(n=65), dict(n=-1), dict(n=1), dict(n=1, counters=(ctypes.c_void_p * 1)()), dict(rows=-1), dict(host=ctypes.create_string_buffer(200))):
        assert norm(**kw) == -1 and b"grad_norm" in lib.benerf_last_error(), kw
    assert norm(room=0) == -2


def test_python_refusals():
    from benerf_amd import _lib, kernels as K, optim
    x = torch.zeros(4)
    with pytest.raises(_lib.BenerfHipError):
        K.AdamWPlan([x], [x.clone()], [x.clone()])
    with pytest.raises(_lib.BenerfHipError):
        K.GradList([x])
    with pytest.raises(ValueError):
        K.GradList([None])
    with pytest.raises(ValueError):
        K.AdamWPlan([], [], [])
    with pytest.raises(ValueError):
        K.grad_norm([x], max_norm=0.0)
    p = torch.nn.Parameter(x.clone())
    for kw in (dict(state_bits=16), dict(max_norm=0.0), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(weight_decay=-1.0), dict(lr=-1.0)):
        with pytest.raises(ValueError):
            optim.FusedAdamW([p], **kw)
    with pytest.raises(NotImplementedError):
        optim.FusedAdamW([p], fused=True)
    p.grad = torch.ones(4)
    with pytest.raises(_lib.BenerfHipError):
        optim.FusedAdamW([p]).step()
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(NotImplementedError):
            optim.FusedAdamW([p], **kw).step()


def test_codec_on_the_host():
    """encode_moment: to nearest on the grid of every block, decode_moment gives the values back; zeros, odd sizes, non-finite values."""
    from benerf_amd import optim
    gen = torch.Generator().manual_seed(3)
    for n in (1, 127, 128, 129, 1000):
        x = torch.randn(n, generator=gen) * torch.exp(3 * torch.randn(n, generator=gen)) * 1e-4
        code, scale = optim.encode_moment(x)
        assert code.dtype == torch.float8_e4m3fn and scale.shape == (-(-n // 128),)
        assert np.array_equal(scale.double().numpy(), O.scale_of(x.double().numpy()))
        back = optim.decode_moment(code, scale).double().numpy()
        s = np.repeat(scale.double().numpy(), 128)[:n]
        # half a step: 2^-4 of the value, or half of 2^-9 scales below the normal range
        assert np.all(np.abs(back - x.double().numpy()) <= np.maximum(2.0 ** -4 * np.abs(x.double().numpy()), 2.0 ** -10 * s))
    code, scale = optim.encode_moment(torch.zeros(5))
    assert not code.float().any() and float(scale) > 0
    bad = torch.tensor([1.0, float("inf"), float("nan"), -2.0])
    back = optim.decode_moment(*optim.encode_moment(bad))
    assert back[0] == 1.0 and back[3] == -2.0 and back[1:3].isnan().all()


def test_oracle_generator():
    """Philox4x32-10 against its authors' published answers (counter and key all zero / all ones / digits of pi)."""
    assert [hex(w) for w in _published(np.array([0, 0, 0, 0]), 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = 0xFFFFFFFF
    assert [hex(w) for w in _published(np.array([ones] * 4), ones, ones)] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]
    assert [hex(w) for w in _published(np.array([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344]), 0xa4093822, 0x299f31d0)] == \
        ["0xd16cfe09", "0x94fdcceb", "0x5001e420", "0x24126ea1"]
    c, t, seed = 0x123456789A, 77, 0x1122334455667788
    ours = O.philox(np.array([c]), t, seed)[0]
    assert list(ours) == list(_published(np.array([c & ones, c >> 32, t, 0x40000000]), seed & ones, seed >> 32))


def _published(ctr, k0, k1):
    v = [int(x) for x in ctr]
    for _ in range(10):
        a, b = v[0] * 0xD2511F53, v[2] * 0xCD9E8D57
        v = [(b >> 32) ^ v[1] ^ k0, b & 0xFFFFFFFF, (a >> 32) ^ v[3] ^ k1, a & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return v


def test_oracle_rounding_is_unbiased():
    """The grid's rounding: exact values stay, the mean over the draws is the value, u > 0 is never 0."""
    r = (np.arange(65536)) / 65536.0
    for y in (1.0, 1.06, 3.3, 0.013, 0.0005, 255.9):
        q = to = O.to_grid(np.full(65536, y), np.ones(65536), r, False)
        step = 2.0 ** (max(np.floor(np.log2(y)), -6) - 3)
        assert abs(q.mean() - y) <= step / 65536 and set(np.unique(to)) <= {step * np.floor(y / step), step * (np.floor(y / step) + 1)}
    assert np.all(O.to_grid(np.full(4, 1e-30), np.ones(4), np.zeros(4), True) == 2.0 ** -9)
    assert np.all(O.to_grid(np.zeros(4), np.ones(4), np.full(4, 0.99), True) == 0)
