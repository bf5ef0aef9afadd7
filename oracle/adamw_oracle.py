"""The optimiser operators over lists (K9) in 64 bits, from their definition (include/benerf_hip.h, csrc/adamw.hip), one tensor at a
time, with bounds on what a 32-bit evaluation may be off by.  numpy only."""
import numpy as np

BLOCK = 128
HALF = 2.0 ** -24                   # a rounding to f32, relative


def philox(counter, t, seed):
    """[len(counter), 4] uint32 words: Philox4x32-10, counter (c, c >> 32, t, 0x40000000), key = seed."""
    c = np.asarray(counter, np.uint64)
    m = np.uint64(0xFFFFFFFF)
    v = [c & m, c >> np.uint64(32), np.full_like(c, t & 0xFFFFFFFF), np.full_like(c, 0x40000000)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = v[0] * np.uint64(0xD2511F53), v[2] * np.uint64(0xCD9E8D57)
        v = [(b >> np.uint64(32)) ^ v[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ v[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(v, 1).astype(np.uint32)


def draws(n, first_block, t, seed):
    """The two 16-bit draws of every element, in [0, 1)."""
    groups = first_block * (BLOCK // 4) + np.arange(-(-n // 4))
    w = philox(groups, t, seed).reshape(-1)[:n]
    return (w & 0xFFFF) / 65536.0, (w >> 16) / 65536.0


def scale_of(x):
    """Power-of-two scale of every block of 128 of |x| (float64)."""
    pad = np.zeros(-(-x.size // BLOCK) * BLOCK)
    pad[:x.size] = np.where(np.isfinite(x), np.abs(x), 0.0)
    top = pad.reshape(-1, BLOCK).max(1)
    e = np.frexp(np.where(top > 0, top, 1.0))[1] - 1
    return np.exp2(np.maximum(np.where(top > 0, e, -100), -100) - 7.0)


def to_grid(x, s, r, keep):
    """Values (not codes) of x rounded to the e4m3 grid of their block with the draw r; s: one scale per element."""
    y = np.abs(x) / s
    e = np.frexp(np.where(y > 0, y, 1.0))[1] - 1
    step = np.exp2(np.maximum(np.where(y > 0, e, -1000), -6) - 3.0)
    q = step * np.floor(y / step + r)
    if keep:
        q = np.where((y > 0) & (q == 0), 2.0 ** -9, q)
    return np.copysign(q * s, x)


def clip_words(grads, max_norm, grad_scale=1.0):
    """(norm, coefficient) over a list of float64 arrays."""
    total = sum(float(np.sum(np.square(g))) for g in grads)
    norm = abs(grad_scale) * np.sqrt(total)
    return norm, min(1.0, max_norm / (norm + 1e-6))


def step(p, g, m, v, lr, t, betas, eps, decay, scale=1.0):
    """One AdamW step in float64.  Returns (p, m, v) and what 32-bit evaluations of them may be off by, element by element.

    Bounds, u = 2^-24: h = g scale has two roundings (scale itself, the product; with a clip coefficient a third): |dh| <= 3 u |h|.
    m + (h - m)(1 - b1): the difference and the product 1 u each, the constant 1 u, the sum 1 u: |dm| <= u (3 |h| (1 - b1) + 3 |h - m|
    (1 - b1) + |m'|) <= 8 u (|h| + |m|).  v b2 + h^2 (1 - b2), all terms positive: 2 u for the first (constant, product), 2 * 3 + 3 u for
    the second, 1 u for the sum: <= 10 u v'.  Root: half of that, and 2 u for a root good to 1 ulp: 7 u.  Denominator: constant, product,
    sum: 10 u.  Quotient and step size: 3 u (division to 1 ulp: 2 u): the step's relative error is 15 u next to that of m.  Weight:
    constant, product, sum: 3 u |p|, and 1 u of the step."""
    b1, b2 = betas
    h = g * scale
    m2 = b1 * m + (1 - b1) * h
    v2 = b2 * v + (1 - b2) * h * h
    den = np.sqrt(v2 / (1 - b2 ** t)) + eps
    move = lr * (m2 / (1 - b1 ** t)) / den
    p2 = (1 - lr * decay) * p - move
    dm = 8 * HALF * (np.abs(h) + np.abs(m))
    # underflow: squares below the smallest f32 vanish, a whole denormal step at most per rounding
    dv = 10 * HALF * v2 + 4 * 2.0 ** -149
    du = 7 * HALF * np.sqrt(v2) + np.sqrt(4 * 2.0 ** -149) * (v2 < 2.0 ** -120)
    dden = np.where(v2 < 2.0 ** -120, np.sqrt(4 * 2.0 ** -149) / np.sqrt(1 - b2 ** t) / den, 0.0)
    dp = 3 * HALF * np.abs(p) + lr / (1 - b1 ** t) * dm / den + (16 * HALF + dden) * np.abs(move)
    return (p2, m2, v2), (dp, dm, dv, du)


def coded_range(x, dx, r, keep):
    """Smallest and largest value that an 8-bit code and its scale may stand for where x is known to +- dx (rounding is monotone; where
    a block's largest value is next to a power of two either scale counts)."""
    lows, highs = [], []
    ax = np.abs(x)
    for s in {tuple(scale_of(np.maximum(ax - dx, 0.0))), tuple(scale_of(ax + dx))}:
        s = np.repeat(np.array(s), BLOCK)[:x.size]
        lows.append(to_grid(np.maximum(ax - dx, 0.0), s, r, False))
        highs.append(to_grid(ax + dx, s, r, keep))
    return np.min(lows, 0), np.max(highs, 0)
