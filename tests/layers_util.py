"""Linear layers, layer norm, dropout and embeddings in NumPy, in 64 bits, for the tests of libgen9blas_llm.so."""
import numpy as np
from scipy.special import erfc

HALF = {np.float16: 2.0 ** -11, np.float32: 2.0 ** -24}      # half a step, relative
TINY = {np.float16: 2.0 ** -25, np.float32: 2.0 ** -149}     # and of a subnormal number


def philox(counter, key):
    """Philox4x32-10 of four arrays of counter words (uint64 holding 32 bits) and two key words."""
    u, low = np.uint64, np.uint64(0xffffffff)
    c = [np.asarray(w, u) for w in counter]
    k = [int(w) for w in key]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & low, (a >> u(32)) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def dropout_factor(rows, cols, p, seed, offset):
    """What dropout multiplies each element by: 0, or the scale."""
    groups = -(-cols // 8)
    c0, c1 = np.broadcast_arrays(np.arange(groups, dtype=np.uint64), np.arange(rows, dtype=np.uint64)[:, None])
    words = philox([c0, c1, np.full_like(c0, offset & 0xffffffff), np.full_like(c0, offset >> 32 & 0xffffffff)], (seed & 0xffffffff, seed >> 32 & 0xffffffff))
    parts = np.stack([w >> np.uint64(s) & np.uint64(0xffff) for w in words for s in (0, 16)], -1).reshape(rows, 8 * groups)[:, :cols]
    limit = round(p * 65536)
    return np.where(parts < limit, 0.0, 65536 / (65536 - limit) if limit < 65536 else 0.0)


def act(z, name):
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        if name == "relu":
            return np.where(z < 0, 0, z)
        if name == "gelu":
            return 0.5 * z * erfc(-z * np.sqrt(0.5))
        if name == "gelu_tanh":
            return z / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))   # 1 + tanh(u) = 2 / (1 + e^-2u), which loses nothing at -u
        return z / (1 + np.exp(-z)) if name == "silu" else z + 0.0


def slope(z, name):
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        if name == "relu":
            return (z > 0).astype(np.float64)
        if name == "gelu":
            return 0.5 * erfc(-z * np.sqrt(0.5)) + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
        if name == "gelu_tanh":
            s = 1 / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
            return s + z * s * (1 - s) * 2 * np.sqrt(2 / np.pi) * (1 + 3 * 0.044715 * z * z)
        if name == "silu":
            s = 1 / (1 + np.exp(-z))
            return s + z * s * (1 - s)
        return np.ones_like(z)


def act_error(z, name, dtype):
    """Rounding of an activation of exact z, relative to its value (its slope also: see there). FP32: the argument of the exponential,
    of size |x|, is off by a few units of 2^-24, which its exponential passes on as |x| of them (GELU: erfc(t) with 2t² = z² of
    them), besides a few units of each function's own. FP16: the hardware's exponential and reciprocal add 2^-20."""
    u, z = 2.0 ** -24, np.clip(z, -100, 100)
    if name in ("silu", "gelu_tanh"):
        x = np.abs(z if name == "silu" else 2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3))
        return (8 + 4 * np.minimum(x, 100)) * u + (2.0 ** -20 if dtype is np.float16 else 0)
    return (16 + 4 * np.minimum(z * z, 200)) * u if name == "gelu" else 0 * z


def layer_norm(x, gamma, beta, eps):
    """y, mean, rstd"""
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    return (x - mean) * rstd * gamma + beta, mean[:, 0], rstd[:, 0]


def layer_norm_back(dy, x, mean, rstd, gamma):
    """dx, dgamma, dbeta"""
    xh, g = (x - mean[:, None]) * rstd[:, None], dy * gamma
    return rstd[:, None] * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True)), (dy * xh).sum(0), dy.sum(0)
