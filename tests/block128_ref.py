"""Plain 64-bit implementations of the block-scaled e4m3 operators (numpy),
and the error bounds the tests hold the kernels to.

A rounding to nearest is off by at most u times the value: u = 2^-24 for
fp32, 2^-8 for bf16; e4m3 by 2^-4 times the value, or half its subnormal step,
2^-10 times the block's scale.  A sum of n fp32 terms in any order is off by
at most n * u32 times the sum of their magnitudes."""

import numpy as np

U32, U16, U8 = 2.0 ** -24, 2.0 ** -8, 2.0 ** -4
UNIT = {"bf16": U16, "f32": U32}


def _table():
    v = []
    for c in range(127):
        e, m = c >> 3, c & 7
        v.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return np.array(v)


E4M3 = _table()  # the 127 finite magnitudes, 0 .. 448
VALUES = np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])


def encode(x):
    """Nearest e4m3 code of each value (ties to the even code), |x| <= 448 or
    not finite; what is not finite becomes 0x7F."""
    a = np.abs(x)
    bad = ~np.isfinite(x)
    a = np.where(bad, 0.0, a)
    hi = np.clip(np.searchsorted(E4M3, a), 1, 126)
    lo = hi - 1
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(x), code | 0x80, code)
    return np.where(bad, 0x7F, code).astype(np.uint8)


def block_top(x, block):
    """Largest finite magnitude of each block of block x 128 values."""
    rows, cols = x.shape
    h, w = -(-rows // block), -(-cols // 128)
    full = np.zeros((h * block, w * 128))
    full[:rows, :cols] = np.where(np.isfinite(x), np.abs(x), 0.0)
    return full.reshape(h, block, w, 128).max(axis=(1, 3))


def scale_bytes(top):
    """E8M0 byte of the smallest power of two s >= 2^-127 with top / s <= 448
    (127 for a block of zeros)."""
    e = np.full(top.shape, -127)
    for k in range(-127, 128):  # by the definition, from below
        e = np.where(top > 448.0 * 2.0 ** k, k + 1, e)
    return np.where(top == 0, 127, e + 127).astype(np.uint8)


def spread(s, rows, cols, block):
    """Each value's scale, as a number."""
    v = np.where(s == 255, np.nan, 2.0 ** (s.astype(np.float64) - 127))
    return v.repeat(block, axis=0)[:rows].repeat(128, axis=1)[:, :cols]


def quantize(x, block):
    s = scale_bytes(block_top(x, block))
    return encode(x / spread(s, *x.shape, block)), s


def restore(q, s, block):
    return VALUES[q] * spread(s, *q.shape, block)


def gemm(qa, sa, qb, sb, block_b):
    """The product, and the same sum over magnitudes."""
    a, b = restore(qa, sa, 1), restore(qb, sb, block_b)
    return a @ b.T, np.abs(a) @ np.abs(b).T


def gemm_bound(ref, mags, k, out):
    """The tensor core adds 32 products at a time to an fp32 accumulator; an
    addition that truncates instead of rounding is off by up to 2 u32, and the
    products' alignment below the largest by as much again: 4 u32 for each
    32 of K, times the sum of magnitudes (a bound on every partial sum).  For
    an fp32 C an accumulator takes 2048 of K, or 2816 where three of 128 tokens
    share 8192, and the parts are added with a rounding each.  Rounded once to
    the output's type."""
    steps = -(-k // 32)
    if out == "f32" and k <= 8192:
        steps = min(steps, 2816 // 32) + -(-k // 2048)
    return 4 * U32 * (steps + 1) * mags + UNIT[out] * np.abs(ref) * (1 + 1e-3) + 1e-300


def norm(h, w, eps):
    rstd = 1.0 / np.sqrt((h * h).mean(axis=1) + eps)
    return rstd, h * rstd[:, None] * w


def norm_backward(dy, h, w, rstd, dh):
    u, g = h * rstd[:, None], dy * w
    mean = (g * u).mean(axis=1, keepdims=True)
    return rstd[:, None] * (g - u * mean) + dh, (dy * u).sum(axis=0)


def sum_steps(cols):
    """Additions that one value meets in the sum over a row: at most 32 within
    a thread (4 chunks of 8), 10 over the warps, and the product's own
    rounding."""
    return 32 + 10 + 1


def rstd_bound(cols):
    # the mean's relative error halves under the root; division, addition of
    # eps, root and reciprocal round once each
    return (sum_steps(cols) / 2 + 4) * U32


def y_bound(cols):
    return rstd_bound(cols) + 2 * U32


def check_quantized(got_q, got_s, y, rel):
    """q, s against values y that the kernel knows to a relative error `rel`:
    the scale is that of a top within the error, and each value is off by at
    most half an e4m3 step under that scale, and y's own error."""
    top = block_top(y, 1)
    assert (got_s >= scale_bytes(top * (1 - rel))).all()
    assert (got_s <= scale_bytes(top * (1 + rel))).all()
    s = spread(got_s, *y.shape, 1)
    err = np.abs(VALUES[got_q] * s - y)
    room = np.maximum(np.abs(y) * U8, s * 2.0 ** -10) * (1 + 1e-6) + 2 * np.abs(y) * rel
    assert (err <= room).all(), (err - room).max()
