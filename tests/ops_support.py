"""Plain 64-bit implementations of the training and 8-bit scoring operators, and how far a kernel may be from them."""
import numpy as np

BLOCK = 128
E4M3 = np.array([m / 8.0 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8.0) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1])  # bytes 0 .. 126


def encode(x):
    """codes [n][blocks * 128] and scale bytes [n][blocks] of float64 rows, from the definition."""
    n, d = x.shape
    blocks = -(-d // BLOCK)
    codes, scales = np.zeros((n, blocks * BLOCK), np.uint8), np.zeros((n, blocks), np.uint8)
    for b in range(blocks):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        finite = np.isfinite(part)
        top = np.where(finite, np.abs(part), 0).max(1)
        for i in range(n):
            power = 0
            if top[i] > 0:
                power = -127
                while top[i] > 448.0 * 2.0 ** power:
                    power += 1
            scales[i, b] = power + 127
            value = np.where(finite[i], np.abs(part[i]), 0) / 2.0 ** power
            hi = np.minimum(np.searchsorted(E4M3, value), len(E4M3) - 1)
            lo = np.maximum(hi - 1, 0)
            near = np.where((value - E4M3[lo] < E4M3[hi] - value) | ((value - E4M3[lo] == E4M3[hi] - value) & (lo % 2 == 0)), lo, hi)
            near = np.where(np.signbit(part[i]), near + 128, near)
            codes[i, b * BLOCK:b * BLOCK + part.shape[1]] = np.where(finite[i], near, 127)
    return codes, scales


def decode(codes, scales, d):
    low = codes & 127
    value = np.where(low == 127, np.nan, E4M3[np.minimum(low, 126)]) * np.where(codes >= 128, -1.0, 1.0)
    return (value.reshape(len(codes), -1, BLOCK) * 2.0 ** (scales.astype(np.float64) - 127)[:, :, None]).reshape(len(codes), -1)[:, :d]


def half_step(dtype):
    """Rounding to `dtype` is off by at most this much of the value."""
    return {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}[dtype]


def softmax(q, v, t, scale, w, dtype):
    """{name: (value, how far off it may be)} of the loss, the lse and both gradients, from float64 inputs.

    Where the bounds come from.  A logit is `scale` times a float32 sum of d exact products (float32 inputs: six times as many, and a part
    of 2^-23 of each product dropped): off by dz = scale (k + 1) 2^-23 sum|q||v|, k the terms (2^-23, not 2^-24: whatever way the matrix unit
    rounds).  Base-2 arithmetic rounds the logit, its product with log2 e and the difference to the maximum: 4 * 2^-24 (|z| + |lse| + 1); the
    exponential and the logarithm are good to 2^-22.  A sum of n positive terms: n 2^-24 of itself at worst.  These add up to de, the relative
    error of a probability and (the sum's) the absolute one of the lse.  g is rounded once (half a step of bf16, or three planes: 2^-23), a
    gradient is a float32 sum of n (or nq) products, in at most 6 partial products for float32, then rounded once."""
    nq, d = q.shape
    n = len(v)
    known = (t >= 0) & (t < n)
    at = np.where(known, t, 0)
    z = scale * (q @ v.T) if n else np.zeros((nq, 0))
    reach = abs(scale) * (np.abs(q) @ np.abs(v).T) if n else np.zeros((nq, 0))
    terms = d if dtype == "bf16" else 6 * d
    if n == 0:
        lse = np.full(nq, -np.inf)
        return {"loss": (np.zeros(nq), np.zeros(nq)), "lse": (lse, np.zeros(nq)), "dq": (np.zeros_like(q), np.zeros_like(q)), "dv": (np.zeros_like(v), np.zeros_like(v))}
    top = z.max(1)
    lse = top + np.log(np.exp(z - top[:, None]).sum(1))
    dz = (terms + 2) * 2.0 ** -23 * reach.max(1) + 4 * 2.0 ** -24 * (np.abs(z).max(1) + np.abs(lse) + 1)
    de = dz + 2.0 ** -21 + n * 2.0 ** -24
    loss = np.where(known, lse - z[np.arange(nq), at], 0)
    p = np.exp(z - lse[:, None])
    hit = np.zeros_like(p)
    hit[np.arange(nq), at] = known
    by = (known * w * scale)[:, None]
    g = (p - hit) * by
    r = half_step(dtype) if dtype == "bf16" else 2.0 ** -23
    # both the logit's own error and the given lse's
    dg = (p * np.expm1(2 * de + dz)[:, None] + 2.0 ** -23 * hit) * np.abs(by)
    dg = dg + r * (np.abs(g) + dg)
    last = half_step(dtype)
    parts = 1 if dtype == "bf16" else 6

    def product(a, da, b, k):
        value = a @ b
        off = da @ np.abs(b) + (parts * k + 2) * 2.0 ** -23 * ((np.abs(a) + da) @ np.abs(b))
        return value, off + last * (np.abs(value) + off)
    return {"loss": (loss, (known * (de + dz)) + 2.0 ** -23 * np.abs(loss)), "lse": (lse, de), "dq": product(g, dg, v, n), "dv": product(g.T, dg.T, q, nq)}


def far(got, want, off):
    """The largest error in units of what is allowed (1 or less is right)."""
    got = np.asarray(got, np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    ratio = np.where(same, 0.0, np.abs(got - want) / np.maximum(off, 1e-300))
    assert not np.isnan(ratio).any()
    return float(ratio.max()) if ratio.size else 0.0
