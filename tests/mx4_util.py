"""MX4 (microscaled 4-bit) matrices in NumPy, in 64 bits, for the tests of libgen9blas_llm.so."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
VALUES = np.concatenate([GRID, -GRID])


def quantize(x):
    """Codes (..., K) and scale bytes (..., ceil(K/32)) of rows of x, by the definition: scale 2^(floor(log2 max|x|) - 2), at
    least 2^-127; nearest value with ties to the even code, beyond 6 to 6; a block with an infinity or NaN has scale 255."""
    x = np.asarray(x, np.float64)
    K = x.shape[-1]
    pad = [(0, 0)] * (x.ndim - 1) + [(0, -K % 32)]
    b = np.pad(x, pad).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    with np.errstate(all="ignore"):
        e = np.where((top > 0) & ~bad, np.frexp(np.where(bad, 1.0, top))[1] - 1, -127 + 2)
    s = np.clip(e - 2 + 127, 0, 254)
    a = np.abs(np.where(bad[..., None], 0, b)) / np.exp2(s - 127.0)[..., None]
    code = np.zeros(a.shape, np.int64)
    for c in range(1, 8):
        mid = (GRID[c - 1] + GRID[c]) / 2
        code = np.where(a >= mid if c % 2 == 0 else a > mid, c, code)
    code += 8 * np.signbit(b)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(*x.shape[:-1], -1)[..., :K].astype(np.uint8), np.where(bad, 255, s).astype(np.uint8)


def values(codes, scales):
    """The values of codes (..., K) with scale bytes (..., ceil(K/32)), float64."""
    K = codes.shape[-1]
    s = np.where(scales == 255, np.nan, np.exp2(np.minimum(scales, 254).astype(np.float64) - 127))
    return VALUES[codes] * np.repeat(s, 32, -1)[..., :K]


def packed(codes):
    """Two codes to a byte, the even one in the low half."""
    c = np.pad(codes, [(0, 0)] * (codes.ndim - 1) + [(0, codes.shape[-1] % 2)])
    return (c[..., 0::2] | c[..., 1::2] << 4).astype(np.uint8)


def sum_bound(K, pieces=3):
    """Rounding of an FP32 sum of K products in chains of 32-product matrix instructions, of which each adds at most two
    units of 2^-24 of a partial sum, over the sum of the magnitudes: `pieces` chains of K/32 steps and a few joins."""
    return (pieces * -(-K // 32) + 16) * 2.0 ** -23


def zero_block_rows(r, K):
    """Codes and scales of 1122 rows (K at least 576) with blocks of zeros, of both signs, under scales of their own: for rows of the largest
    scales 0, 60, 100, 120 and 130 every scale from there to 254, in the second and the eighteenth block; rows of zeros with each
    scale 0..254; and two rows with a NaN block (scale 255), of codes zero and others."""
    n = -(-K // 32)
    rows = [(e, s) for e in (0, 60, 100, 120, 130) for s in range(e, 255)]
    e, s = np.array(rows).T
    codes = r.integers(0, 16, (len(rows), K)).astype(np.uint8)
    codes[:, 0] |= 1                                       # no accident leaves the row's largest block empty
    scales = np.maximum(e[:, None] - r.integers(0, 4, (len(rows), n)), 0)
    scales[:, 0] = e
    for b in (1, 17):
        codes[:, 32 * b:32 * b + 32] &= 8
        scales[:, b] = s
    zeros = 8 * r.integers(0, 2, (255, K))
    nan, nan_scales = codes[-2:].copy(), scales[-2:].copy()
    nan[0, 64:96] = 0
    nan_scales[:, 2] = 255
    return (np.concatenate([codes, zeros, nan]).astype(np.uint8),
            np.concatenate([scales, np.repeat(np.arange(255)[:, None], n, 1), nan_scales]).astype(np.uint8))
