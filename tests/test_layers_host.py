"""The tests' own references of dropout and of gradients, and what the entry points say without a GPU."""
import ctypes
import os

import numpy as np
import pytest

from layers_util import act, dropout_factor, layer_norm, layer_norm_back, philox, slope

ROOT = os.path.dirname(os.path.dirname(os.path.realpath(__file__)))


def test_philox_known_answers():
    """The generator's published answers for counters and keys of zeros, of ones, and of digits of pi."""
    for counter, key, want in (((0,) * 4, (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
                               ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
                               ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        assert tuple(int(w) for w in philox(counter, key)) == want


def test_dropout_factor():
    f = dropout_factor(3, 20, 0.5, 1, 2)
    assert f.shape == (3, 20) and set(f.ravel()) == {0.0, 2.0}
    assert np.array_equal(f[:, :13], dropout_factor(3, 13, 0.5, 1, 2)) and np.array_equal(f[:2], dropout_factor(2, 20, 0.5, 1, 2))
    assert (dropout_factor(2, 9, 1.0, 1, 2) == 0).all() and (dropout_factor(2, 9, 0.0, 1, 2) == 1).all()


@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu", "none"])
def test_slopes(name):
    z = np.linspace(-8, 8, 1001) + 1e-4
    h = 1e-6
    assert np.allclose((act(z + h, name) - act(z - h, name)) / (2 * h), slope(z, name), atol=1e-8)
    assert np.abs(slope(z, name)).max() <= 1.13


def test_layer_norm_gradients():
    r = np.random.default_rng(0)
    x, dy, gamma, beta = r.normal(0, 1, (3, 7)), r.normal(0, 1, (3, 7)), r.normal(1, 0.3, 7), r.normal(0, 1, 7)
    _, mean, rstd = layer_norm(x, gamma, beta, 1e-3)
    for v, g in zip((x, gamma, beta), layer_norm_back(dy, x, mean, rstd, gamma)):
        for i in np.ndindex(v.shape):
            old, loss = v[i], []
            for s in (1e-5, -1e-5):
                v[i] = old + s
                loss.append((layer_norm(x, gamma, beta, 1e-3)[0] * dy).sum())
            v[i] = old
            assert abs((loss[0] - loss[1]) / 2e-5 - g[i]) < 1e-7


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="a GPU is present: the no-device path is not reachable")
def test_no_device_status():
    L = ctypes.CDLL(os.path.join(ROOT, "gen9-gpu-blas_amd", "libgen9blas_llm.so"))
    L.gen9blas_llm_error.restype = ctypes.c_char_p
    p, d, f, u = ctypes.c_void_p(None), ctypes.c_double(0), ctypes.c_float(1), ctypes.c_uint64(0)
    for rc in (L.gen9blas_linear(1, 1, 1, 1, p, 1, p, 1, p, 0, p, 0, d, u, u, p, 0, p, 1),
               L.gen9blas_linear_backward(1, 1, 1, 1, p, 1, p, 0, 0, d, u, u, p, 1, p, 1, p, 1, p, 1, p, 0),
               L.gen9blas_layer_norm(1, 1, 1, p, 1, p, p, f, p, 1, p), L.gen9blas_layer_norm_backward(1, 1, 1, p, 1, p, 1, p, p, p, 1, p, p, 0),
               L.gen9blas_dropout(1, 1, 1, p, 1, d, u, u, p, 0, p, 1), L.gen9blas_embedding(1, 1, 1, 1, p, 1, p, 8, f, p, 1),
               L.gen9blas_embedding_backward(1, 1, 1, 1, p, 1, p, 8, f, 1, p, 1, 0)):
        assert rc == -5 and L.gen9blas_llm_last_status() == -5 and L.gen9blas_llm_error()
