"""Linear layers, layer norm, dropout and embeddings (libgen9blas_llm.so) on a GPU, against 64-bit NumPy.

Bounds. A sum of n products in FP32 is off by at most n units of 2^-24 of the sum of their magnitudes, in whatever order it is
taken; a result is rounded once, by half a step of its type (tests/layers_util.py has these, and what activations add). Where
a bound has a number of operations in it, it is counted in the test."""
import numpy as np
import pytest

from layers_util import HALF, TINY, act, act_error, dropout_factor, layer_norm, layer_norm_back, slope

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [np.float16, np.float32]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def gpu(torch, x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def laid(torch, x, pad, shift):
    """x (2-D) on the GPU in rows of `pad` elements more, beginning `shift` elements into a buffer that is NaN everywhere else."""
    rows, cols = x.shape
    buf = torch.full((shift + rows * (cols + pad) + 8,), float("nan"), dtype=torch.float16 if x.dtype == np.float16 else torch.float32, device="cuda")
    view = buf[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    view.copy_(torch.from_numpy(np.ascontiguousarray(x)))
    return view, buf


def untouched(torch, view, buf):
    """Whether all of buf but the view is still NaN."""
    inside = torch.zeros(buf.shape, dtype=torch.bool, device="cuda")
    rows, cols = view.shape
    first = (view.data_ptr() - buf.data_ptr()) // buf.element_size()
    for r in range(rows):
        inside[first + r * view.stride(0):first + r * view.stride(0) + cols] = True
    return bool(torch.isnan(buf[~inside]).all())


def near(got, want, bound, dtype):
    """|got - want| <= bound and one rounding to dtype; infinities and NaN alike."""
    got = got.cpu().numpy() if hasattr(got, "cpu") else got
    assert got.dtype == dtype and got.shape == want.shape
    got = got.astype(np.float64)
    fine = np.isfinite(want) & (np.abs(want) + bound < np.finfo(dtype).max)
    err = np.abs(got - want)[fine]
    limit = (bound + (np.abs(want) + bound) * HALF[dtype] + TINY[dtype])[fine] if np.ndim(bound) else bound + (np.abs(want[fine]) + bound) * HALF[dtype] + TINY[dtype]
    assert (err <= limit).all(), (float((err / limit).max()), int((err > limit).sum()), got.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want))


# ---- linear ----
def linear64(x, w, b, name, R, factor):
    """y, z and the bound of z's error: K products and one addition."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    z = x @ w.T + (0 if b is None else b.astype(np.float64))
    dz = (x.shape[1] + 1) * U * (np.abs(x) @ np.abs(w).T + (0 if b is None else np.abs(b)))
    y = act(z, name) * factor
    # the steepest activation has a slope of 1.13; the scale, its product and the residual's sum are three roundings
    bound = (1.13 * dz + np.abs(act(z, name)) * act_error(z, name, x.dtype.type)) * factor + 3 * U * np.abs(y)
    if R is not None:
        y = y + R.astype(np.float64)
        bound = bound + U * np.abs(y)
    return y, z, bound, dz


def check_linear(g9, torch, dtype, M, N, K, name="none", bias=True, residual=False, save=False, p=0.0, seed=0, pad=0, shift=0):
    r = np.random.default_rng(M + 7 * N + 31 * K)
    x, w = r.normal(0, 1, (M, K)).astype(dtype), (r.normal(0, 1, (N, K)) / np.sqrt(K)).astype(dtype)
    b = r.normal(0, 0.5, N).astype(np.float32) if bias else None
    R = r.normal(0, 1, (M, N)).astype(dtype) if residual else None
    offset = (5 << 32) + M
    factor = dropout_factor(M, N, p, seed, offset) if p else np.ones((M, N))
    y, z, bound, dz = linear64(x, w, b, name, R, factor)
    if dtype is np.float16:
        bound = bound + np.abs(act(z, name)) * factor * 2.0 ** -20    # act_error's part of FP16
    X, W = laid(torch, x, pad, shift)[0], laid(torch, w, pad, shift)[0]
    res = None if R is None else laid(torch, R, pad, shift)[0]
    C, cbuf = laid(torch, np.zeros((M, N), dtype), pad, shift)
    Z, zbuf = laid(torch, np.zeros((M, N), dtype), pad, shift) if save else (None, None)
    out = g9.linear(X, W, bias=None if b is None else gpu(torch, b), act=name, dropout=p, seed=seed, offset=offset, residual=res, Z=Z, C=C)
    assert out is C
    near(C, y, bound, dtype)
    if p:
        assert np.array_equal(C.cpu().numpy().astype(np.float64)[factor == 0], (np.zeros((M, N)) if R is None else R.astype(np.float64))[factor == 0])
    assert untouched(torch, C, cbuf)
    if save:
        near(Z, z, dz, dtype)
        assert untouched(torch, Z, zbuf)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 500, 300), (2, 33, 64), (3, 70, 256), (4, 16, 512), (5, 9, 7), (8, 100, 768), (9, 31, 1000), (16, 17, 256),
                                   (17, 1, 1), (17, 100, 63), (18, 64, 64), (33, 65, 65), (64, 64, 128), (100, 300, 250), (129, 257, 31), (200, 130, 1030),
                                   (257, 520, 96), (1000, 24, 333), (20, 2048, 4096)])
def test_linear(g9, torch_dev, dtype, M, N, K):
    check_linear(g9, torch_dev, dtype, M, N, K, bias=True)
    check_linear(g9, torch_dev, dtype, M, N, K, "gelu", bias=M % 2 == 0, residual=True, save=True, p=0.3, seed=(9 << 32) + 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,N,K", [(3, 90, 300), (80, 90, 300)])
@pytest.mark.parametrize("residual,save,p", [(False, False, 0.0), (True, True, 0.0), (False, True, 0.25), (True, False, 1.0)])
def test_linear_forms(g9, torch_dev, dtype, name, M, N, K, residual, save, p):
    check_linear(g9, torch_dev, dtype, M, N, K, name, residual=residual, save=save, p=p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 4, 12, 40, 300])
@pytest.mark.parametrize("pad,shift", [(1, 0), (3, 1), (8, 1), (2, 2), (5, 3)])
def test_linear_strides(g9, torch_dev, dtype, M, pad, shift):
    check_linear(g9, torch_dev, dtype, M, 75, 256, "silu", residual=True, save=True, p=0.1, pad=pad, shift=shift)
    check_linear(g9, torch_dev, dtype, M, 64, 40, "none", residual=True, pad=pad, shift=shift)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(2304, 2048, 512), (1200, 1500, 1024), (700, 5000, 192), (48, 4096, 4096), (600, 1100, 3000), (4000, 520, 130)])
def test_linear_tiles(g9, torch_dev, dtype, M, N, K):
    """Sizes that take each of the tile kernels; on small integers every sum is exact, so the results are too."""
    torch = torch_dev
    r = np.random.default_rng(M)
    x, w = r.integers(-2, 3, (M, K)).astype(dtype), r.integers(-1, 2, (N, K)).astype(dtype)
    b, R = r.integers(-3, 4, N).astype(np.float32), r.integers(-3, 4, (M, N)).astype(dtype)
    z = x.astype(np.float64) @ w.astype(np.float64).T + b
    C, Z = g9.linear(gpu(torch, x), gpu(torch, w), gpu(torch, b), "relu", residual=gpu(torch, R), Z=(Z := torch.empty(M, N, dtype=torch.float16 if dtype is np.float16 else torch.float32, device="cuda"))), Z
    assert np.abs(z).max() < 2048
    assert np.array_equal(Z.cpu().numpy(), z.astype(dtype)) and np.array_equal(C.cpu().numpy(), (np.maximum(z, 0) + R).astype(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(3, 8300, 4090), (8, 8200, 4224), (12, 2100, 4100), (16, 8193, 4352), (17, 4100, 8320), (24, 5000, 8000), (32, 8256, 4100), (33, 3000, 2817),
                                   (40, 9000, 3900), (47, 2100, 4096), (64, 2050, 4224), (64, 8300, 1100), (30, 34000, 1000), (20, 90000, 100), (20, 170000, 200)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (2, 2), (3, 1)])
def test_linear_of_some_rows(g9, torch_dev, dtype, M, N, K, pad, shift):
    """Large weights under few rows: whole and cut pieces of k, columns that end inside a workgroup's."""
    check_linear(g9, torch_dev, dtype, M, N, K, "silu", residual=True, save=pad > 0, pad=pad, shift=shift)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ACTS)
def test_activations_over_their_range(g9, torch_dev, dtype, name):
    """Z straight from the bias: every size of argument, both zeros, infinities and NaN (which ReLU keeps, too)."""
    torch = torch_dev
    z = np.concatenate([s * np.exp2(np.arange(-40, 14, 0.25)) for s in (1, -1)] + [np.arange(-30, 30, 0.03125), [0.0, -0.0, np.inf, -np.inf, np.nan]]).astype(np.float32)
    N = len(z)
    want = act(z.astype(np.float64), name)
    bound = np.nan_to_num(np.abs(want) * (act_error(np.nan_to_num(z.astype(np.float64)), name, dtype) + 2 * U))
    for M in (2, 20):
        x, w = torch.zeros(M, 64, device="cuda"), torch.zeros(N, 64, device="cuda")
        if dtype is np.float16:
            x, w = x.half(), w.half()
        Y = g9.linear(x, w, gpu(torch, z), name).cpu().numpy()
        for row in Y:
            fine = np.isfinite(z)
            # the factor of z, 1 / (1 + e^-x) or erfc / 2, may be 0 where it is below 2^-126: |z| of that are lost
            near(row[fine], want[fine], bound[fine] + np.abs(z.astype(np.float64))[fine] * 2.0 ** -126, dtype)
        assert np.isnan(Y[:, -1]).all() and np.isposinf(Y[:, -3]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,N,K,p", [(1, 1, 1, 0.0), (1, 70, 300, 0.2), (7, 33, 65, 0.0), (50, 130, 90, 0.4), (300, 75, 64, 0.1), (600, 2500, 40, 0.0)])
def test_linear_backward(g9, torch_dev, dtype, name, M, N, K, p):
    torch = torch_dev
    r = np.random.default_rng(M + N)
    dy, z, x, w = (r.normal(0, 1, s).astype(dtype) for s in ((M, N), (M, N), (M, K), (N, K)))
    seed, offset = 77, 1 << 40
    f = dropout_factor(M, N, p, seed, offset) if p else 1.0
    s, z64 = slope(z.astype(np.float64), name), z.astype(np.float64)
    g = dy.astype(np.float64) * f * s
    # a slope is a sum of two terms, each with its activation's relative error (three for the product of two); dropout's
    # scale and the products round three times; the rounding to the type is half a step
    terms = {"gelu": 1, "relu": 1, "none": 1}.get(name, 1 + 3 * np.abs(z64))
    eg = np.abs(dy * f) * (terms * 3 * act_error(z64, name, dtype) + 3 * U * np.abs(s)) + 3 * U * np.abs(g)
    eq = eg + HALF[dtype] * (np.abs(g) + eg) + TINY[dtype] if name != "none" or p else 0 * g
    g9x, g9w = x.astype(np.float64), w.astype(np.float64)
    Z = gpu(torch, z) if name != "none" else None
    dX, dW, db = g9.linear_backward(gpu(torch, dy), gpu(torch, x), gpu(torch, w), Z=Z, act=name, dropout=p, seed=seed, offset=offset)
    near(dX, g @ g9w, eq @ np.abs(g9w) + (N + 1) * U * (np.abs(g) @ np.abs(g9w)), dtype)
    near(dW, g.T @ g9x, eq.T @ np.abs(g9x) + (M + 1) * U * (np.abs(g).T @ np.abs(g9x)), dtype)
    near(db, g.sum(0), eg.sum(0) + (M + 1) * U * np.abs(g).sum(0), np.float32)
    # added to what is there, and only what is asked for
    dW2, db2 = gpu(torch, np.ones((N, K), dtype)), gpu(torch, np.ones(N, np.float32))
    got = g9.linear_backward(gpu(torch, dy), gpu(torch, x), gpu(torch, w), Z=Z, act=name, dropout=p, seed=seed, offset=offset, dW=dW2, db=db2, accumulate=True, grads="wb")
    assert got[0] is None and got[1] is dW2 and got[2] is db2
    near(dW2, 1 + g.T @ g9x, eq.T @ np.abs(g9x) + (M + 2) * U * (1 + np.abs(g).T @ np.abs(g9x)), dtype)
    near(db2, 1 + g.sum(0), eg.sum(0) + (M + 2) * U * (1 + np.abs(g).sum(0)), np.float32)
    only = g9.linear_backward(gpu(torch, dy), gpu(torch, x), gpu(torch, w), Z=Z, act=name, dropout=p, seed=seed, offset=offset, grads="x")
    assert only[1] is None and only[2] is None and torch.equal(only[0], dX)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ACTS)
def test_what_is_dropped_is_zero(g9, torch_dev, dtype, name):
    """Infinities and NaN in places that dropout takes, forward and backward: zeros are left of them, in the gradients too."""
    torch = torch_dev
    M, N, K, p, seed, offset = 40, 72, 64, 0.5, 3, 9
    t = torch.float16 if dtype is np.float16 else torch.float32
    lost = torch.from_numpy(dropout_factor(M, N, p, seed, offset) == 0).cuda()
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=t, device="cuda").repeat(M * N // 3).view(M, N)
    x, w = torch.eye(K, dtype=t, device="cuda")[:M], torch.ones(N, K, dtype=t, device="cuda")
    good = torch.ones(M, N, dtype=t, device="cuda")
    z = torch.where(lost, bad, good)
    for rows in (1, 3, 12, M):                     # a bias that is bad where the first row is dropped
        b = torch.where(lost[0], bad[0], good[0]).float()
        y = g9.linear(torch.zeros(rows, K, dtype=t, device="cuda"), w, b, name, p, seed, offset)[0]
        assert torch.isfinite(y).all() and (y[lost[0]] == 0).all()
    for dy in (torch.where(lost, bad, good), good):
        got = g9.linear_backward(dy, x, w, Z=z if name != "none" else None, act=name, dropout=p, seed=seed, offset=offset)
        want = g9.linear_backward(good, x, w, Z=good if name != "none" else None, act=name, dropout=p, seed=seed, offset=offset)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_relu_clips_has_no_gradient(g9, torch_dev, dtype):
    """Infinities and NaN of dY where Z is not above zero; a NaN of Z passes dY on."""
    torch = torch_dev
    M, N, K = 33, 70, 64
    t = torch.float16 if dtype is np.float16 else torch.float32
    z = torch.tensor([1.0, -1.0, 0.0, -float("inf"), float("inf")], dtype=t, device="cuda").repeat(M * N // 5).view(M, N)
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=t, device="cuda").repeat(M * N // 3).view(M, N)
    x, w = torch.eye(K, dtype=t, device="cuda")[:M], torch.ones(N, K, dtype=t, device="cuda")
    got = g9.linear_backward(torch.where(z > 0, torch.ones_like(z), bad), x, w, Z=z, act="relu")
    want = g9.linear_backward((z > 0).to(t), x, w)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    _, _, db = g9.linear_backward(torch.ones_like(z), x, w, Z=torch.full_like(z, float("nan")), act="relu")
    assert (db == M).all()


@pytest.mark.parametrize("name", ACTS[1:])
def test_linear_gradients_against_differences(g9, torch_dev, name):
    """Central differences of the framework's own forward pass in FP32: a step h = 2^-6 leaves h²/6 of the third derivative (at most 4
    for these activations, with sums of 12 terms of weights below 1) and 2 roundings of 2^-22 over 2h."""
    torch = torch_dev
    r = np.random.default_rng(5)
    M, N, K, h = 3, 5, 12, 2.0 ** -6
    x, w, b, dy = (gpu(torch, r.uniform(-0.6, 0.6, s).astype(np.float32)) for s in ((M, K), (N, K), (N,), (M, N)))
    x.abs_().add_(0.05)   # ReLU: away from its corner
    w.abs_().add_(0.05)
    b.abs_().add_(0.05)
    Z = torch.empty(M, N, device="cuda")
    g9.linear(x, w, b, name, 0.2, 3, 4, Z=Z)
    grads = g9.linear_backward(dy, x, w, Z, name, 0.2, 3, 4)

    def loss():
        return float((g9.linear(x, w, b, name, 0.2, 3, 4).double() * dy.double()).sum())

    for v, g in zip((x, w, b), grads):
        for i in range(v.numel()):
            flat, old = v.view(-1), float(v.view(-1)[i])
            flat[i] = old + h
            up, hi = loss(), float(flat[i])
            flat[i] = old - h
            down, lo = loss(), float(flat[i])
            flat[i] = old
            assert abs((up - down) / (hi - lo) - float(g.view(-1)[i])) <= h * h / 6 * 4 * 15 + 15 * 2.0 ** -22 / h


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_backward_without_rows(g9, torch_dev, dtype):
    torch = torch_dev
    t = torch.float16 if dtype is np.float16 else torch.float32
    dy, x, w = (torch.empty(s, dtype=t, device="cuda") for s in ((0, 33), (0, 20), (33, 20)))
    dW, db = torch.full((33, 24), 5.0, dtype=t, device="cuda")[:, :20], torch.full((33,), 5.0, device="cuda")
    dX, *_ = g9.linear_backward(dy, x, w, dW=dW, db=db, accumulate=True)
    assert dX.shape == (0, 20) and (dW == 5).all() and (db == 5).all()
    g9.linear_backward(dy, x, w, Z=dy, act="gelu", dW=dW, db=db)
    assert (dW == 0).all() and (db == 0).all() and (dW._base[:, 20:] == 5).all()
    assert g9.linear(x, w).shape == (0, 33)


# ---- layer norm ----
def check_norm(g9, torch, x, gamma, beta, eps=1e-5, pad=0, shift=0):
    dtype = x.dtype.type
    M, N = x.shape
    r = np.random.default_rng(N)
    X = laid(torch, x, pad, shift)[0]
    Y, ybuf = laid(torch, np.zeros((M, N), dtype), pad, shift)
    stats = torch.empty(M, 2, device="cuda")
    g, b = (None if v is None else gpu(torch, v) for v in (gamma, beta))
    out = g9.layer_norm(X, g, b, eps=eps, out=Y, stats=stats)
    assert out is Y and untouched(torch, Y, ybuf)
    g64, b64 = np.ones(N) if gamma is None else gamma.astype(np.float64), np.zeros(N) if beta is None else beta.astype(np.float64)
    x64 = x.astype(np.float64)
    y, mean, rstd = layer_norm(x64, g64, b64, eps)
    size = np.abs(x64).mean(1)
    # sums of N terms in FP32: the mean is off by em, which comes off again up to its own rounding (against the spread: ed); the
    # variance by as many units of itself, half of which its root passes on
    n = N + 8
    em = n * U * size
    spread = np.abs(x64 - mean[:, None])
    ed = 4 * U * np.abs(mean) + n * U * (spread.mean(1) + em)
    ev = n * U + 2 * ed * rstd + (ed * rstd) ** 2
    near(Y, y, (ed * rstd)[:, None] * np.abs(g64) + np.abs(y - b64) * (ev[:, None] + 8 * U) + 2 * U * (np.abs(y) + np.abs(b64)), dtype)
    s = stats.cpu().numpy().astype(np.float64)
    assert (np.abs(s[:, 0] - mean) <= ed + 2 * U * np.abs(mean)).all() and (np.abs(s[:, 1] - rstd) <= rstd * (ev + 4 * U)).all()
    # the gradients, from these stats
    dy = r.normal(0, 1, (M, N)).astype(dtype)
    dx, dg, db = layer_norm_back(dy.astype(np.float64), x64, s[:, 0], s[:, 1], g64)
    xh, gy = np.abs((x64 - s[:, :1]) * s[:, 1:]), np.abs(dy * g64)
    exh = 3 * U * (np.abs(x64) + np.abs(s[:, :1])) * s[:, 1:]
    a, c = gy.mean(1, keepdims=True), (gy * xh).mean(1, keepdims=True)
    bound = s[:, 1:] * (n * U * a + xh * n * U * c + exh * c + xh * (gy * exh).mean(1, keepdims=True) + 8 * U * (gy + a + xh * c))
    dY = laid(torch, dy, pad, shift)[0]
    DX, dbuf = laid(torch, np.zeros((M, N), dtype), pad, shift)
    got = g9.layer_norm_backward(dY, X, stats, g, dX=DX)
    near(DX, dx, bound, dtype)
    assert untouched(torch, DX, dbuf)
    dabs = np.abs(dy.astype(np.float64))
    bg, bb = (M + 4) * U * (dabs * xh).sum(0) + (dabs * exh).sum(0), (M + 4) * U * dabs.sum(0)
    near(got[1], dg, bg, np.float32)
    near(got[2], db, bb, np.float32)
    more = g9.layer_norm_backward(dY, X, stats, g, dgamma=torch.ones(N, device="cuda"), dbeta=torch.ones(N, device="cuda"), accumulate=True, grads="gb")
    assert more[0] is None
    near(more[1], 1 + dg, bg + U * (1 + np.abs(dg)), np.float32)
    near(more[2], 1 + db, bb + U * (1 + np.abs(db)), np.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(1, 1), (3, 2), (2, 7), (5, 63), (4, 64), (300, 65), (33, 500), (7, 512), (70, 1000), (2, 1024), (1, 4096), (9, 4097), (600, 300),
                                 (5, 8192), (3, 8200), (2, 16384), (2, 20001), (1, 40000), (2, 70001)])
def test_layer_norm(g9, torch_dev, dtype, M, N):
    r = np.random.default_rng(M * N)
    x = (r.normal(0, 1, (M, N)) * np.exp(r.normal(0, 0.5, N)) + r.normal(0, 1, (M, 1))).astype(dtype)
    check_norm(g9, torch_dev, x, (1 + r.normal(0, 0.3, N)).astype(np.float32), r.normal(0, 0.3, N).astype(np.float32))
    check_norm(g9, torch_dev, x, None, None, eps=0.1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [60, 256, 999, 3000, 9001])
@pytest.mark.parametrize("pad,shift", [(1, 0), (8, 1), (3, 3)])
def test_layer_norm_strides(g9, torch_dev, dtype, N, pad, shift):
    r = np.random.default_rng(N)
    x = r.normal(0.5, 2, (37, N)).astype(dtype)
    check_norm(g9, torch_dev, x, r.normal(1, 0.3, N).astype(np.float32), r.normal(0, 0.3, N).astype(np.float32), pad=pad, shift=shift)


@pytest.mark.parametrize("N", [100, 4096, 20000])
def test_layer_norm_of_rows_far_from_zero(g9, torch_dev, N):
    """Means of up to 2^14 times the spread (FP32): what x holds of the spread is not lost to the mean's rounding."""
    r = np.random.default_rng(N)
    x = (np.array([[2.0 ** 14], [-300.0], [0.0], [7.0 * 2 ** 10]]) + r.normal(0, 1, (4, N))).astype(np.float32)
    check_norm(g9, torch_dev, x, None, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 48, 1000, 5000, 30000])
def test_layer_norm_special_rows(g9, torch_dev, dtype, N):
    """Rows of one value (no variance), of zeros, and with infinities and NaN, which stay in their rows."""
    torch = torch_dev
    r = np.random.default_rng(N)
    x = r.normal(0, 1, (9, N)).astype(dtype)
    x[1], x[2], x[4, N // 2], x[5, N - 1], x[7, 0] = 0, 3, np.inf, np.nan, -np.inf
    beta = r.normal(0, 1, N).astype(np.float32)
    stats = torch.empty(9, 2, device="cuda")
    y = g9.layer_norm(gpu(torch, x), None, gpu(torch, beta), stats=stats).cpu().numpy()
    assert np.array_equal(y[1], beta.astype(dtype)) and np.array_equal(y[2], beta.astype(dtype))
    assert np.isnan(y[[4, 5, 7]]).all() and np.isfinite(y[[0, 3, 6, 8]]).all()
    alone = g9.layer_norm(gpu(torch, x[[0, 3, 6, 8]]), None, gpu(torch, beta)).cpu().numpy()
    assert np.array_equal(alone, y[[0, 3, 6, 8]])
    assert (stats[1:3, 1] - 1e-5 ** -0.5).abs().max() < 1e-3


def test_layer_norm_without_rows(g9, torch_dev):
    torch = torch_dev
    x, stats = torch.empty(0, 20, device="cuda"), torch.empty(0, 2, device="cuda")
    assert g9.layer_norm(x).shape == (0, 20)
    dx, dg, db = g9.layer_norm_backward(x, x, stats)
    assert dx.shape == (0, 20) and (dg == 0).all() and (db == 0).all() and dg.shape == db.shape == (20,)


# ---- dropout ----
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(1, 1), (1, 7), (3, 8), (5, 9), (100, 64), (33, 1001), (2, 100000), (5000, 3)])
@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 0.999, 1.0])
def test_dropout(g9, torch_dev, dtype, M, N, p):
    torch = torch_dev
    r = np.random.default_rng(M + N)
    x, R = r.normal(0, 1, (M, N)).astype(dtype), r.normal(0, 1, (M, N)).astype(dtype)
    seed, offset = (1 << 63) + 12345, (7 << 32) + 3
    f = dropout_factor(M, N, p, seed, offset)
    y = x.astype(np.float64) * f
    got = g9.dropout(gpu(torch, x), p, seed, offset)
    near(got, y, 2 * U * np.abs(y), dtype)     # the scale's rounding and the product's
    assert (got.cpu().numpy()[f == 0] == 0).all()
    for pad, shift in ((0, 0), (3, 1)):
        out, buf = laid(torch, np.zeros((M, N), dtype), pad, shift)
        g9.dropout(laid(torch, x, pad, shift)[0], p, seed, offset, residual=laid(torch, R, pad, shift)[0], out=out)
        near(out, y + R, 2 * U * np.abs(y) + U * np.abs(y + R), dtype)
        assert untouched(torch, out, buf)


def test_dropout_masks(g9, torch_dev):
    """Infinities and NaN that are dropped are gone; another seed, offset or row has another mask; the share is p's."""
    torch = torch_dev
    x = torch.full((512, 1000), float("nan"), device="cuda")
    f = dropout_factor(512, 1000, 0.25, 1, 2)
    assert np.array_equal(torch.isnan(g9.dropout(x, 0.25, 1, 2)).cpu().numpy(), f > 0)
    x.fill_(float("inf"))
    assert np.array_equal(torch.isinf(g9.dropout(x, 0.25, 1, 2)).cpu().numpy(), f > 0)
    x.fill_(1)
    masks = [(g9.dropout(x, 0.25, *s) != 0).float() for s in ((1, 2), (1, 3), (2, 2), (1 + (1 << 32), 2), (1, 2 + (1 << 32)))]
    for i, a in enumerate(masks):
        # 512000 independent elements: five deviations of their mean are 5 sqrt(p (1 - p) / n)
        assert abs(float(a.mean()) - 0.75) < 5 * (0.25 * 0.75 / 512000) ** 0.5
        for b in masks[:i]:
            assert abs(float((a * b).mean()) - 0.75 ** 2) < 5 * (0.75 ** 2 * (1 - 0.75 ** 2) / 512000) ** 0.5


# ---- embeddings ----
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 1000, 4096), (7, 5, 3), (100, 300, 64), (33, 50, 129), (1000, 10, 1000), (5, 100000, 8)])
@pytest.mark.parametrize("wide", [np.int32, np.int64])
def test_embedding(g9, torch_dev, dtype, T, V, D, wide):
    torch = torch_dev
    r = np.random.default_rng(T + V)
    table, ids = r.normal(0, 1, (V, D)).astype(dtype), r.integers(0, V, T).astype(wide)
    if T > 6:
        ids[[1, 3, 5]] = -1, V, np.iinfo(wide).min
        ids[6] = np.iinfo(wide).max
    ok = (ids >= 0) & (ids < V)
    want = np.where(ok[:, None], table[np.where(ok, ids, 0)].astype(np.float64), 0)
    assert np.array_equal(g9.embedding(gpu(torch, table), gpu(torch, ids)).cpu().numpy(), want.astype(dtype))
    for pad, shift in ((3, 1), (8, 0)):
        out, buf = laid(torch, np.zeros((T, D), dtype), pad, shift)
        g9.embedding(laid(torch, table, pad, shift)[0], gpu(torch, ids), scale=3.7, out=out)
        near(out, want * 3.7, 2 * U * np.abs(want * 3.7), dtype)     # the scale as FP32, and the product
        assert untouched(torch, out, buf)


def embedding_grad(dy, ids, V):
    s, a = np.zeros((V, dy.shape[1])), np.zeros((V, dy.shape[1]))
    ok = (ids >= 0) & (ids < V)
    np.add.at(s, ids[ok], dy[ok].astype(np.float64))
    np.add.at(a, ids[ok], np.abs(dy[ok].astype(np.float64)))
    return s, a


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (3, 1, 5), (31, 40, 8), (32, 2, 100), (33, 1, 64), (64, 3, 2049), (100, 255, 33), (1000, 256, 16), (1023, 257, 24), (1025, 65535, 9), (5000, 65536, 4),
                                   (5000, 70, 130), (40000, 300, 20), (3000, 1 << 17, 12), (9, (1 << 20) + 100, 4), (5000, 1 << 18, 8), (1100, 200, 1500), (4096, 40, 257)])
def test_embedding_backward(g9, torch_dev, dtype, T, V, D):
    torch = torch_dev
    r = np.random.default_rng(T + V)
    dy = r.normal(0, 1, (T, D)).astype(dtype)
    ids = np.minimum((V * r.random(T) ** 3).astype(np.int64), V - 1)     # some far more often than others
    if T > 30:
        ids[r.integers(0, T, 5)] = [-1, V, -(1 << 40), 1 << 40, np.iinfo(np.int64).max]
    want, size = embedding_grad(dy, ids, V)
    bound = (T + 2) * U * size
    got = g9.embedding_backward(gpu(torch, dy), gpu(torch, ids), V)
    near(got, want, bound, dtype)
    assert torch.equal(got, g9.embedding_backward(gpu(torch, dy), gpu(torch, ids), V))     # bit for bit
    out, buf = laid(torch, np.ones((V, D), dtype), 5, 3)
    g9.embedding_backward(laid(torch, dy, 3, 1)[0], gpu(torch, ids), V, scale=0.5, out=out, accumulate=True)
    near(out, 1 + 0.5 * want, bound + U * (1 + np.abs(want)), dtype)
    assert untouched(torch, out, buf) and (out[torch.from_numpy(size.sum(1) == 0).cuda()] == 1).all()
    f32 = torch.full((V, D), float("nan"), device="cuda")
    assert g9.embedding_backward(gpu(torch, dy), gpu(torch, np.clip(ids, -1, V).astype(np.int32)), V, out=f32) is f32
    near(f32, want, bound, np.float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_backward_is_exact_on_integers(g9, torch_dev, dtype):
    """Every token in its row, none twice: 20000 tokens in runs of 1 to 5000, small integers."""
    torch = torch_dev
    r = np.random.default_rng(1)
    ids = np.concatenate([np.full(5000, 17), np.full(33, 3), np.full(64, 16), np.full(2000, 18), r.integers(0, 700, 12903)])
    r.shuffle(ids)
    dy = r.integers(-1, 2, (len(ids), 72)).astype(dtype)
    want, _ = embedding_grad(dy, ids, 700)
    assert np.array_equal(g9.embedding_backward(gpu(torch, dy), gpu(torch, ids), 700).cpu().numpy(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,D", [(1, 1), (15, 8), (17, 70), (64, 72), (65, 300), (2000, 33), (10000, 900)])
@pytest.mark.parametrize("T", [1, 2, 63, 64, 257, 1023, 1024])
def test_embedding_backward_of_few_tokens(g9, torch_dev, dtype, T, V, D):
    """Small integers, whose sums are exact: one token in all places, tokens in turn, and a few places of others among one's."""
    torch = torch_dev
    r = np.random.default_rng(T)
    one = np.full(T, V // 2)
    some = one.copy()
    some[r.integers(0, T, 1 + T // 10)] = r.integers(-2, V + 2, 1 + T // 10)
    for ids in (one, np.arange(T) * 7 % V, some):
        dy = r.integers(-1, 2, (T, D)).astype(dtype)
        want, _ = embedding_grad(dy, ids, V)
        i = gpu(torch, ids)
        out, buf = laid(torch, np.full((V, D), 7, dtype), 3, 1)
        g9.embedding_backward(gpu(torch, dy), i, V, out=out)
        assert np.array_equal(out.cpu().numpy(), want)
        beside = buf[1:1 + V * (D + 3)].view(V, D + 3)[:, D:]
        assert torch.isnan(beside).all() and torch.isnan(buf[:1]).all() and torch.isnan(buf[1 + V * (D + 3):]).all()
        assert np.array_equal(g9.embedding_backward(gpu(torch, dy), i, V, out=torch.ones(V, D, device="cuda"), accumulate=True).cpu().numpy(), 1 + want)


def test_embedding_empty(g9, torch_dev):
    torch = torch_dev
    ids, dy = torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, 6, device="cuda")
    assert g9.embedding(torch.ones(4, 6, device="cuda"), ids).shape == (0, 6)
    out = torch.ones(4, 6, device="cuda")
    g9.embedding_backward(dy, ids, 4, out=out, accumulate=True)
    assert (out == 1).all()
    assert (g9.embedding_backward(dy, ids, 4, out=out) == 0).all()
    none = torch.full((3000,), -1, device="cuda")
    assert (g9.embedding_backward(torch.ones(3000, 6, device="cuda"), none, 4, out=out) == 0).all()


# ---- together ----
@pytest.mark.parametrize("M", [6, 70])
def test_a_training_step(g9, torch_dev, M):
    """Embedding, norm, two linear layers with dropout and residual, and an output layer on the embedding's table, forward and
    backward in FP32, against torch's gradients of the same in 64 bits on the CPU. A value passes through five sums of at most
    260 terms each way: 2 · 5 · 260 units of 2^-24, on values that a norm keeps near one, with a factor of 8 for the weights."""
    torch = torch_dev
    gen = torch.Generator().manual_seed(M)
    V, D, F, p = 260, 64, 200, 0.2
    E, W1, W2 = (torch.randn(s, generator=gen) * k for s, k in (((V, D), 0.3), ((F, D), D ** -0.5), ((D, F), F ** -0.5)))
    b1, b2, g, b, g2, bb2 = (torch.randn(n, generator=gen) * 0.1 + c for n, c in ((F, 0), (D, 0), (D, 1), (D, 0), (D, 1), (D, 0)))
    ids, target = torch.randint(0, V, (M,), generator=gen), torch.randn(M, V, generator=gen)
    params = [E, W1, b1, W2, b2, g, b, g2, bb2]
    keep = torch.from_numpy(dropout_factor(M, D, p, 5, 6))
    d = [t.double().requires_grad_() for t in params]
    ln = torch.nn.functional.layer_norm
    x = d[0][ids] * 2.0
    y = x + keep * (torch.nn.functional.gelu(ln(x, (D,), d[5], d[6]) @ d[1].t() + d[2]) @ d[3].t() + d[4])
    (ln(y, (D,), d[7], d[8]) @ d[0].t() * target.double()).sum().backward()

    E, W1, b1, W2, b2, g, b, g2, bb2 = (t.cuda() for t in params)
    ids, target = ids.cuda(), target.cuda()
    new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    s1, s2, Z = new(M, 2), new(M, 2), new(M, F)
    x = g9.embedding(E, ids, 2.0)
    n1 = g9.layer_norm(x, g, b, stats=s1)
    h = g9.linear(n1, W1, b1, "gelu", Z=Z)
    y = g9.linear(h, W2, b2, dropout=p, seed=5, offset=6, residual=x)
    n2 = g9.layer_norm(y, g2, bb2, stats=s2)
    g9.linear(n2, E)
    dn2, dE, _ = g9.linear_backward(target, n2, E, grads="xw")
    dy, dg2, dbb2 = g9.layer_norm_backward(dn2, y, s2, g2)
    dh, dW2, db2 = g9.linear_backward(dy, h, W2, dropout=p, seed=5, offset=6)
    dn1, dW1, db1 = g9.linear_backward(dh, n1, W1, Z=Z, act="gelu")
    dx, dg, db = g9.layer_norm_backward(dn1, x, s1, g)
    g9.embedding_backward(dx + dy, ids, V, 2.0, out=dE, accumulate=True)
    for got, want in zip((dE, dW1, db1, dW2, db2, dg, db, dg2, dbb2), d):
        want = want.grad
        assert (got.cpu().double() - want).abs().max() <= 8 * 2 * 5 * 260 * U * max(1, float(want.abs().max()))


def test_captured_and_replayed(g9, torch_dev):
    """A graph of the operators that need no work buffers (a token through embedding, norm, linear layers and dropout), replayed on
    new tokens with other work between; those that need some are refused, and the capture can be left."""
    torch = torch_dev
    V, D, F = 300, 512, 2048
    gen = torch.Generator().manual_seed(5)
    table, w1, w2 = (torch.randn(s, generator=gen).half().cuda() / 8 for s in ((V, D), (F, D), (D, F)))
    gamma, bias = torch.rand(D, generator=gen).cuda(), torch.randn(F, generator=gen).cuda()
    ids = torch.tensor([7], device="cuda")

    def step():
        e = g9.embedding(table, ids, scale=2.0)
        h = g9.linear(g9.layer_norm(e, gamma), w1, bias, act="silu")
        return g9.dropout(g9.linear(h, w2, residual=e), 0.25, seed=3, offset=4)

    big = torch.randn(4096, D, generator=gen).half().cuda()
    before = g9.linear(big, w1, bias)
    g9.set_nowait(True)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
        for token in (7, 0, 299, -1, 8):
            ids.fill_(token)
            graph.replay()
            got = y.clone()
            g9.linear(big, w1, bias)                                       # other work, and another residual stream's buffers
            g9.embedding_backward(big, torch.arange(4096, device="cuda") % V, V)
            assert torch.equal(got, step()), token
            torch.cuda.synchronize()
        dy, tokens = torch.randn(4096, F, generator=gen).half().cuda(), torch.arange(4096, device="cuda") % V
        for call in (lambda: g9.linear_backward(dy, big, w1), lambda: g9.embedding_backward(big, tokens, V),
                     lambda: g9.layer_norm_backward(big, big, torch.ones(4096, 2, device="cuda"))):
            refused = torch.cuda.CUDAGraph()
            with torch.cuda.graph(refused):
                with pytest.raises(RuntimeError, match="captured"):
                    call()
    finally:
        g9.set_nowait(False)
    assert torch.equal(g9.linear(big, w1, bias), before)


def test_gradients_captured_and_replayed(g9, torch_dev):
    """A graph of the gradients that need no work buffers: few tokens' tables, few rows' norms."""
    torch = torch_dev
    V, D, T = 500, 320, 600
    gen = torch.Generator().manual_seed(6)
    dy, x = (torch.randn(T, D, generator=gen).cuda() for _ in range(2))
    ids, stats = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.empty(4, 2, device="cuda")
    table, total = torch.empty(V, D, device="cuda"), torch.zeros(V, D, device="cuda")

    def step(table, total):
        g9.embedding_backward(dy, ids, V, out=table)
        g9.embedding_backward(dy, ids, V, out=total, accumulate=True)
        g9.layer_norm(x[:4], stats=stats)
        return g9.layer_norm_backward(dy[:4], x[:4], stats)

    g9.set_nowait(True)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(table, total)
        for seed in range(4):
            ids.copy_(torch.randint(-1, V if seed % 2 else 2, (T,), generator=gen))
            x.mul_(-1.5)
            want = torch.empty_like(table), total.clone()
            graph.replay()
            norm = step(*want)
            for a, b in zip((table, total, *got), (*want, *norm)):
                assert torch.equal(a, b), seed
            torch.cuda.synchronize()
    finally:
        g9.set_nowait(False)


def test_calls_that_wait_are_not_captured(g9, torch_dev):
    torch = torch_dev
    x = torch.randn(3, 40, device="cuda")
    want = g9.layer_norm(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(RuntimeError, match="set_nowait"):
            g9.layer_norm(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x + 1) and torch.equal(g9.layer_norm(x), want)


def test_counters_of_other_integer_types(g9, torch_dev):
    torch = torch_dev
    x = torch.ones(5, 40, device="cuda")
    want = g9.dropout(x, 0.5, seed=-1, offset=1 << 40)
    assert torch.equal(g9.dropout(x, 0.5, seed=np.int64(-1), offset=np.int64(1 << 40)), want)
    with pytest.raises(TypeError):
        g9.dropout(x, 0.5, seed=1.5)


def test_streams(g9, torch_dev):
    """Calls from another torch stream are ordered with it on both sides; in no-wait mode too."""
    torch = torch_dev
    side = torch.cuda.Stream()
    w, ids = torch.eye(512, device="cuda"), torch.arange(512, device="cuda")
    try:
        g9.set_nowait(True)
        with torch.cuda.stream(side):
            x = torch.zeros(300, 512, device="cuda")
            for i in range(20):
                x = g9.dropout(g9.linear(x + 1, w, residual=x), 0.0)
                x = x - g9.embedding(w, ids)[:300] + g9.embedding_backward(torch.ones(512, 512, device="cuda"), ids, 512)[:300] - 1 + w[:300]
            want = torch.full_like(x, 2.0 ** 20 - 1)
            assert torch.equal(x, want)
    finally:
        g9.set_nowait(False)
    torch.cuda.synchronize()


def test_host_operands(g9, torch_dev):
    """NumPy arrays go to the GPU and back; float64 and bfloat16 become float32."""
    torch = torch_dev
    r = np.random.default_rng(0)
    x, w = r.integers(-2, 3, (5, 12)).astype(np.float64), r.integers(-2, 3, (7, 12)).astype(np.float64)
    y = g9.linear(x, w, np.ones(7))
    assert isinstance(y, np.ndarray) and y.dtype == np.float32 and np.array_equal(y, x @ w.T + 1)
    assert isinstance(g9.linear_backward(y, x, w)[1], np.ndarray)
    assert isinstance(g9.layer_norm(x), np.ndarray) and isinstance(g9.dropout(x, 0.5), np.ndarray)
    assert np.array_equal(g9.embedding(w, [3, -1, 0])[[0, 2]], w[[3, 0]])
    assert np.array_equal(g9.embedding_backward(x, np.array([1, 1, 0, 2, 2], np.uint8), 3), [x[2], x[0] + x[1], x[3] + x[4]])
    b = torch.from_numpy(x).cuda().bfloat16()
    assert torch.equal(g9.linear(b, torch.from_numpy(w).cuda().bfloat16()).cpu().double(), torch.from_numpy(x @ w.T))


# ---- refusals ----
def test_refusals(g9, torch_dev):
    torch = torch_dev
    f = lambda *s: torch.ones(s, device="cuda")  # noqa: E731
    x, w = f(4, 8), f(6, 8)
    for error, call in [
            (ValueError, lambda: g9.linear(x, f(6, 9))), (TypeError, lambda: g9.linear(x, w.half())), (ValueError, lambda: g9.linear(x, w, f(5))),
            (ValueError, lambda: g9.linear(x, w, act="swish")), (RuntimeError, lambda: g9.linear(x, w, dropout=1.5)), (RuntimeError, lambda: g9.linear(x, w, dropout=float("nan"))),
            (RuntimeError, lambda: g9.linear(x, w, dropout=-0.1)), (ValueError, lambda: g9.linear(x, w, residual=f(4, 7))), (TypeError, lambda: g9.linear(x, w, residual=f(4, 6).half())),
            (ValueError, lambda: g9.linear(x, w, C=f(6, 4).t())), (ValueError, lambda: g9.linear(x, w, Z=f(4, 6).half())), (ValueError, lambda: g9.linear(x, w, C=f(4, 7))),
            (RuntimeError, lambda: g9.linear(x, w, C=f(1, 6).expand(4, 6))), (RuntimeError, lambda: g9.linear(f(4, 0), f(6, 0))), (ValueError, lambda: g9.linear(f(8), w)),
            (ValueError, lambda: g9.linear_backward(f(4, 6), x, w, act="silu")), (ValueError, lambda: g9.linear_backward(f(4, 5), x, w)),
            (ValueError, lambda: g9.linear_backward(f(4, 6), x, w, accumulate=True)), (ValueError, lambda: g9.linear_backward(f(4, 6), x, w, grads="y")),
            (TypeError, lambda: g9.linear_backward(f(4, 6).half(), x, w)), (ValueError, lambda: g9.linear_backward(f(4, 6), x, w, db=f(5))),
            (ValueError, lambda: g9.layer_norm(x, f(9))), (RuntimeError, lambda: g9.layer_norm(x, eps=-1.0)), (RuntimeError, lambda: g9.layer_norm(x, eps=float("nan"))),
            (ValueError, lambda: g9.layer_norm(x, stats=f(4, 3))), (ValueError, lambda: g9.layer_norm(x, stats=f(4, 4)[:, ::2])), (ValueError, lambda: g9.layer_norm(x, out=f(4, 9))),
            (RuntimeError, lambda: g9.layer_norm(f(4, 0))), (ValueError, lambda: g9.layer_norm_backward(x, f(4, 9), f(4, 2))), (ValueError, lambda: g9.layer_norm_backward(x, x, f(3, 2))),
            (ValueError, lambda: g9.layer_norm_backward(x, x, f(4, 2), accumulate=True)), (RuntimeError, lambda: g9.dropout(x, 1.01)), (ValueError, lambda: g9.dropout(x, 0.5, residual=f(4, 9))),
            (ValueError, lambda: g9.dropout(x, 0.5, out=f(4, 9))), (TypeError, lambda: g9.embedding(w, f(3))), (ValueError, lambda: g9.embedding(w, torch.zeros(2, 2, dtype=torch.int64))),
            (TypeError, lambda: g9.embedding(w, torch.zeros(2, dtype=torch.bool))), (ValueError, lambda: g9.embedding_backward(x, torch.zeros(3, dtype=torch.int64), 5)),
            (ValueError, lambda: g9.embedding_backward(x, torch.zeros(4, dtype=torch.int64), 5, out=f(5, 8).half())), (ValueError, lambda: g9.embedding_backward(x, torch.zeros(4, dtype=torch.int64), 5, accumulate=True)),
            (RuntimeError, lambda: g9.embedding(f(0, 8), torch.zeros(3, dtype=torch.int64)))]:
        with pytest.raises(error):
            call()


def test_another_device_is_refused(g9, torch_dev, monkeypatch):
    """Operands on another GPU than the library's, as if it had opened the second one."""
    torch = torch_dev
    f = lambda *s: torch.ones(s, device="cuda")  # noqa: E731
    g9.linear(f(2, 8), f(3, 8))
    monkeypatch.setattr(g9, "_llm_device", g9._llm_device + 1)
    for call in (lambda: g9.linear(f(2, 8), f(3, 8)), lambda: g9.linear_backward(f(2, 3), f(2, 8), f(3, 8)), lambda: g9.layer_norm(f(2, 8)), lambda: g9.layer_norm_backward(f(2, 8), f(2, 8), f(2, 2)),
                 lambda: g9.dropout(f(2, 8), 0.5), lambda: g9.embedding(f(4, 8), torch.zeros(2, dtype=torch.int64, device="cuda")),
                 lambda: g9.embedding_backward(f(2, 8), torch.zeros(2, dtype=torch.int64, device="cuda"), 4)):
        with pytest.raises(ValueError, match="library runs on"):
            call()


def test_c_refusals(g9, torch_dev):
    """The C entry points: host memory, NULL and operands that run past their allocation, wrong sizes, unknown types."""
    torch = torch_dev
    L = g9._llm_library()
    BAD, NOT = -3, -2
    x, o = torch.ones(64, 64, device="cuda"), torch.ones(64, 64, device="cuda")
    d, e, memory = x.data_ptr(), o.data_ptr(), np.ones((64, 64), np.float32)
    host = memory.ctypes.data
    big = 1 << 30     # rows that no allocation of this process has
    linear = lambda **k: L.gen9blas_linear(*{**dict(type=1, M=4, N=4, K=4, X=d, ldx=64, W=d, ldw=64, bias=None, act=0, Z=None, ldz=0, p=0.0, seed=0, offset=0, R=None, ldr=0, Y=e, ldy=64), **k}.values())  # noqa: E731
    assert linear(M=0) == 0 and linear(N=0) == 0
    for k in (dict(X=host), dict(W=None), dict(Y=host), dict(R=host, ldr=64), dict(Z=host, ldz=64), dict(bias=host), dict(ldx=3), dict(ldw=3), dict(ldy=3), dict(R=d, ldr=3), dict(Z=d, ldz=3), dict(K=0),
              dict(p=2.0), dict(M=big, ldx=4, ldy=4)):
        assert linear(**k) == BAD and L.gen9blas_llm_error() and L.gen9blas_llm_last_status() == BAD, k
    for k in (dict(type=2), dict(type=3), dict(act=5), dict(act=-1), dict(K=1 << 22, ldx=1 << 22, ldw=1 << 22), dict(M=0x7fffffff), dict(N=0x7ffffff0, ldy=0x7fffffff)):
        assert linear(**k) == NOT, k
    back = lambda **k: L.gen9blas_linear_backward(*{**dict(type=1, M=4, N=4, K=4, dY=d, lddy=64, Z=d, ldz=64, act=2, p=0.0, seed=0, offset=0, X=d, ldx=64, W=d, ldw=64, dX=None, lddx=0, dW=None, lddw=0, db=None, acc=0), **k}.values())  # noqa: E731
    assert back() == 0 and back(dX=e, lddx=64, X=None) == 0 and back(dW=e, lddw=64, W=None) == 0 and back(db=e, X=None, W=None) == 0
    for k in (dict(dX=e, lddx=3), dict(dX=host, lddx=64), dict(dW=e, lddw=64, X=None), dict(dX=e, lddx=64, W=host), dict(db=host), dict(db=e, Z=None), dict(db=e, dY=host), dict(db=e, lddy=3), dict(db=e, p=-1.0)):
        assert back(**k) == BAD, k
    norm = lambda **k: L.gen9blas_layer_norm(*{**dict(type=1, M=4, N=4, X=d, ldx=64, g=None, b=None, eps=0.1, Y=e, ldy=64, stats=None), **k}.values())  # noqa: E731
    nback = lambda **k: L.gen9blas_layer_norm_backward(*{**dict(type=1, M=4, N=4, dY=d, lddy=64, X=d, ldx=64, stats=d, g=None, dX=e, lddx=64, dg=None, db=None, acc=0), **k}.values())  # noqa: E731
    drop = lambda **k: L.gen9blas_dropout(*{**dict(type=1, M=4, N=4, X=d, ldx=64, p=0.5, seed=0, offset=0, R=None, ldr=0, Y=e, ldy=64), **k}.values())  # noqa: E731
    emb = lambda **k: L.gen9blas_embedding(*{**dict(type=1, T=4, V=4, D=4, table=d, ldt=64, ids=d, w=8, scale=1.0, Y=e, ldy=64), **k}.values())  # noqa: E731
    eback = lambda **k: L.gen9blas_embedding_backward(*{**dict(type=1, T=4, V=4, D=4, dY=d, lddy=64, ids=d, w=8, scale=1.0, ot=1, dT=e, lddt=64, acc=0), **k}.values())  # noqa: E731
    for call, bad, refused in (
            (norm, [dict(X=host), dict(Y=None), dict(g=host), dict(b=host), dict(stats=host), dict(N=0), dict(ldx=3), dict(ldy=3), dict(eps=-1.0), dict(M=big, ldx=4, ldy=4)], [dict(type=3)]),
            (nback, [dict(dY=host), dict(X=host), dict(stats=None), dict(dX=host), dict(dg=host), dict(db=host), dict(lddx=3), dict(lddy=3), dict(N=0)], [dict(type=2)]),
            (drop, [dict(X=host), dict(Y=None), dict(R=host, ldr=64), dict(R=d, ldr=3), dict(p=1.1), dict(ldx=3), dict(ldy=3)], [dict(type=-1)]),
            (emb, [dict(table=host), dict(ids=host), dict(Y=host), dict(V=0), dict(ldt=3), dict(ldy=3), dict(T=big, ldy=4)], [dict(type=2), dict(w=2)]),
            (eback, [dict(dY=host), dict(ids=None), dict(dT=host), dict(lddy=3), dict(lddt=3), dict(V=big, lddt=4)], [dict(type=2), dict(ot=0), dict(w=1)])):
        for k in bad:
            assert call(**k) == BAD and L.gen9blas_llm_error(), k
        for k in refused:
            assert call(**k) == NOT, k
    assert nback(dX=None) == 0 and drop(M=0) == 0 and emb(T=0) == 0 and eback(V=0) == 0
    g9.flush()
    assert (x == 1).all()
