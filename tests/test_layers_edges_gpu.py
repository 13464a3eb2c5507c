"""Linear layers, layer norm, dropout and embeddings (libgen9blas_llm.so) on a GPU, beyond tests/test_layers_gpu.py: rows far from
zero backward, overflows and infinities, matrices laid oddly, and the loops that only long inputs enter. Against 64-bit NumPy, with
that file's bounds: n units of 2^-24 for a sum of n products in any order, half a step for a result's rounding."""
import numpy as np
import pytest

from layers_util import HALF, TINY, dropout_factor, layer_norm, layer_norm_back, slope
from test_layers_gpu import U, check_norm, embedding_grad, gpu, laid, near, untouched

pytestmark = pytest.mark.gpu
DTYPES = [np.float16, np.float32]


def tensor_type(torch, dtype):
    return torch.float16 if dtype is np.float16 else torch.float32


# ---- the gradients of a linear layer ----
def gradients64(dy, z, x, w, name, f):
    """dX, dW, db and their bounds for dy, z, x, w of one type: dZ's own error is counted in test_linear_backward of
    tests/test_layers_gpu.py; here z is None (dZ = dy) or the activation is ReLU, whose slope is exact."""
    dtype = dy.dtype.type
    g = dy.astype(np.float64) * f * (1 if z is None else slope(z.astype(np.float64), name))
    # dropout's scale and its product
    eg = 2 * U * np.abs(g) if np.ndim(f) else 0 * g
    eq = eg + HALF[dtype] * (np.abs(g) + eg) + TINY[dtype] if np.ndim(f) else 0 * g
    x, w = x.astype(np.float64), w.astype(np.float64)
    M, N = g.shape
    return ((g @ w, eq @ np.abs(w) + (N + 1) * U * (np.abs(g) @ np.abs(w))), (g.T @ x, eq.T @ np.abs(x) + (M + 1) * U * (np.abs(g).T @ np.abs(x))),
            (g.sum(0), eg.sum(0) + (M + 1) * U * np.abs(g).sum(0)))


@pytest.mark.parametrize("M,N,K", [(4096, 520, 264), (300, 4096, 1032), (8, 4096, 4096)])
@pytest.mark.parametrize("name", ["none", "gelu"])
def test_linear_backward_repeats_itself(g9, torch_dev, M, N, K, name):
    """Bit for bit, with other work between the calls."""
    torch = torch_dev
    gen = torch.Generator(device="cuda").manual_seed(M)
    dy, z, x, w = (torch.randn(s, generator=gen, device="cuda").half() for s in ((M, N), (M, N), (M, K), (N, K)))
    call = lambda: g9.linear_backward(dy, x, w, Z=z if name != "none" else None, act=name)  # noqa: E731
    first = [v.clone() for v in call()]
    for i in range(4):
        g9.linear_backward(dy * -3, x, w)
        g9.linear(x, w)
        for a, b in zip(call(), first):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("M,N,K", [(300, 520, 264), (150, 131, 1029)])
def test_linear_backward_rounds_dz_and_no_more(g9, torch_dev, M, N, K):
    """FP16: with a slope and a scale that leave dZ as it is (ReLU, half of it dropped), dX and dW are the products of the exact dZ but
    for their FP32 sums and one rounding; and those of a dropped share of 0.3 are the products of dZ rounded once."""
    torch = torch_dev
    r = np.random.default_rng(M)
    dy, z, x, w = (r.normal(0, 1, s).astype(np.float16) for s in ((M, N), (M, N), (M, K), (N, K)))
    for p in (0.5, 0.3):
        f = dropout_factor(M, N, p, 3, 4)
        scaled = (dy.astype(np.float32) * f.astype(np.float32)).astype(np.float16)   # FP32 product, rounded once
        want = gradients64(scaled, z, x, w, "relu", 1.0)
        got = g9.linear_backward(gpu(torch, dy), gpu(torch, x), gpu(torch, w), Z=gpu(torch, z), act="relu", dropout=p, seed=3, offset=4)
        near(got[0], *want[0], np.float16)
        near(got[1], *want[1], np.float16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name,p", [("none", 0.0), ("relu", 0.0), ("relu", 0.25)])
@pytest.mark.parametrize("M,N,K", [(5, 70, 33), (130, 131, 150), (200, 64, 129), (64, 300, 257)])
@pytest.mark.parametrize("pad,shift", [(1, 0), (2, 1), (3, 1), (8, 3)])
def test_linear_backward_strides(g9, torch_dev, dtype, name, p, M, N, K, pad, shift):
    """Every operand and result in rows of its own stride and alignment: odd ones of FP16, which long products copy first."""
    torch = torch_dev
    r = np.random.default_rng(M + N + K)
    dy, z, x, w = (r.normal(0, 1, s).astype(dtype) for s in ((M, N), (M, N), (M, K), (N, K)))
    f = dropout_factor(M, N, p, 5, 6) if p else 1.0
    want = gradients64(dy, z if name != "none" else None, x, w, name, f)
    DY, Z, X, W = (laid(torch, v, pad, shift)[0] for v in (dy, z, x, w))
    for old in (False, True):
        (DX, xbuf), (DW, wbuf) = laid(torch, np.zeros((M, K), dtype), pad, shift), laid(torch, np.full((N, K), 1.0 if old else 0.0, dtype), pad, shift)
        db = torch.full((N,), 1.0 if old else 7.0, device="cuda")
        g9.linear_backward(DY, X, W, Z=Z if name != "none" else None, act=name, dropout=p, seed=5, offset=6, dX=DX, dW=DW, db=db, accumulate=old)
        near(DX, *want[0], dtype)
        near(DW, want[1][0] + old, want[1][1] + 2 * U * (old + np.abs(want[1][0])), dtype)
        near(db, want[2][0] + old, want[2][1] + 2 * U * (old + np.abs(want[2][0])), np.float32)
        assert untouched(torch, DX, xbuf) and untouched(torch, DW, wbuf)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(5000, 75, 24), (40000, 40, 16)])
def test_linear_backward_of_many_rows(g9, torch_dev, dtype, M, N, K):
    """More than 64 rows in a block of the first pass, and more than 64 blocks."""
    torch = torch_dev
    r = np.random.default_rng(M)
    dy, z, x, w = (r.normal(0, 1, s).astype(dtype) for s in ((M, N), (M, N), (M, K), (N, K)))
    f = dropout_factor(M, N, 0.2, 7, 8)
    want = gradients64(dy, z, x, w, "relu", f)
    got = g9.linear_backward(gpu(torch, dy), gpu(torch, x), gpu(torch, w), Z=gpu(torch, z), act="relu", dropout=0.2, seed=7, offset=8)
    near(got[0], *want[0], dtype)
    near(got[1], *want[1], dtype)
    near(got[2], *want[2], np.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_at_infinity(g9, torch_dev, dtype, name):
    """Pre-activations past FP16's range are stored as infinities: the slope there is that of the end, 0 or 1, as it is next to
    them; a NaN stays one."""
    torch = torch_dev
    t = tensor_type(torch, dtype)
    ends = [-np.inf, np.inf, -60000.0, 60000.0] + ([] if dtype is np.float16 else [-3e38, 3e38, -1e20, 1e20])
    z = torch.tensor(ends, dtype=t, device="cuda").repeat(40, 16)
    M, N = z.shape
    dy = torch.arange(-M * N // 2, M * N // 2, device="cuda").view(M, N).remainder(17).to(t) + 1
    x, w = torch.ones(M, 64, dtype=t, device="cuda"), torch.eye(N, 64, dtype=t, device="cuda")
    dX, dW, db = g9.linear_backward(dy, x, w, Z=z, act=name)
    want = torch.where(z > 0, dy, torch.zeros_like(dy))
    assert torch.equal(dX, (want.double() @ w.double()).to(t)) and torch.equal(db, want.float().sum(0)) and torch.equal(dW, want.double().sum(0).to(t)[:, None].expand(N, 64))
    z[3, 5] = float("nan")
    assert torch.isnan(g9.linear_backward(dy, x, w, Z=z, act=name, grads="b")[2][5]) == (name != "relu")   # ReLU's passes dY on


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_pre_activations_past_fp16_train(g9, torch_dev, name):
    """A forward pass that is finite though Z is not has finite gradients."""
    torch = torch_dev
    x, w = torch.ones(40, 64, device="cuda").half(), torch.ones(70, 64, device="cuda").half()
    bias = torch.full((70,), -1e5, device="cuda")
    Z = torch.empty(40, 70, device="cuda", dtype=torch.float16)
    y = g9.linear(x, w, bias, name, Z=Z)
    assert torch.isneginf(Z).all() and (y == 0).all()
    for g in g9.linear_backward(torch.ones_like(y), x, w, Z=Z, act=name):
        assert (g == 0).all()


def test_columns_past_one_launch(g9, torch_dev):
    """More columns than a launch of 1024 threads for 64 of them can have."""
    torch = torch_dev
    N = (1 << 28) + 77
    dy = torch.randint(-9, 10, (2, N), dtype=torch.int8, device="cuda").half()
    w, x = torch.zeros(N, 1, dtype=torch.float16, device="cuda"), torch.zeros(2, 1, dtype=torch.float16, device="cuda")
    db = torch.full((N,), float("nan"), device="cuda")
    g9.linear_backward(dy, x, w, db=db, grads="b")
    assert torch.equal(db, dy[0].float() + dy[1].float())
    del dy, w, x, db
    torch.cuda.empty_cache()


# ---- results past FP16's range ----
def same(torch, got, want):
    """Equal in every element, infinities with their signs."""
    assert np.array_equal(got.cpu().numpy(), want), (got.cpu().numpy()[got.cpu().numpy() != want][:5], want[got.cpu().numpy() != want][:5])


@pytest.mark.parametrize("M", [1, 4, 12, 40, 300])
@pytest.mark.parametrize("K", [64, 256, 4096])
def test_overflows_of_linear(g9, torch_dev, M, K):
    """Z and Y straight from the bias, around FP16's largest numbers: 65504 holds up to 65520, past which results are infinite; a residual
    is added before the rounding."""
    torch = torch_dev
    b = np.array([s * v for s in (1, -1) for v in (65504, 65519.9, 65520, 65536, 1e5, 3e38, np.inf, 65503, 1, 0)] * 5, np.float32)
    N = len(b)
    x, w = torch.zeros(M, K, device="cuda").half(), torch.zeros(N, K, device="cuda").half()
    with np.errstate(over="ignore"):
        rows = np.broadcast_to(b.astype(np.float16), (M, N))
        Z = torch.empty(M, N, dtype=torch.float16, device="cuda")
        same(torch, g9.linear(x, w, gpu(torch, b), Z=Z), rows)
        same(torch, Z, rows)
        R = np.broadcast_to(np.clip(-b, -60000, 60000).astype(np.float16), (M, N))
        same(torch, g9.linear(x, w, gpu(torch, b), residual=gpu(torch, R)), (b + R.astype(np.float32)).astype(np.float16))
        f = dropout_factor(M, N, 0.5, 1, 2).astype(np.float32)
        same(torch, g9.linear(x, w, gpu(torch, b), dropout=0.5, seed=1, offset=2), np.where(f > 0, b * 2, 0).astype(np.float16))


def test_overflows_of_sums_and_scales(g9, torch_dev):
    """Of dropout's scale, of a table's rows and their gradients, and of a norm's gamma: signed infinities, and finite where the FP32 sum is."""
    torch = torch_dev
    v = np.array([40000, -40000, 32760, -32760, 65504, -65504, 1, 0], np.float16)
    x = np.broadcast_to(np.tile(v, 5), (33, 40))
    with np.errstate(over="ignore"):
        f = dropout_factor(33, 40, 0.5, 5, 6).astype(np.float32)
        same(torch, g9.dropout(gpu(torch, x), 0.5, 5, 6), (x * f).astype(np.float16))
        same(torch, g9.dropout(gpu(torch, x), 0.5, 5, 6, residual=gpu(torch, -x)), (x * f - x).astype(np.float16))
        same(torch, g9.embedding(gpu(torch, x), gpu(torch, np.array([3, 0])), scale=2.0), (x[:2].astype(np.float32) * 2).astype(np.float16))
        for T in (2, 3, 2000, 5000):     # each of the sort's forms
            ids, dy = np.where(np.arange(T) < 3, 1, 2), np.zeros((T, 40), np.float16)
            dy[:2] = x[:2]
            dy[2:3] = np.sign(x[:1]) * -30000
            total = dy[:3].astype(np.float32).sum(0)
            got = g9.embedding_backward(gpu(torch, dy), gpu(torch, ids), 4)
            same(torch, got[1], total.astype(np.float16))
            assert (got[[0, 2, 3]] == 0).all()
            same(torch, g9.embedding_backward(gpu(torch, dy), gpu(torch, ids), 4, out=torch.empty(4, 40, device="cuda"))[1], total)
        for N in (40, 1000, 33000):
            row = np.where(np.arange(N) % 2, 1.0, -1.0).astype(np.float16)[None]
            y = g9.layer_norm(gpu(torch, row), torch.full((N,), 1e6, device="cuda"))
            same(torch, y, np.where(row > 0, np.inf, -np.inf).astype(np.float16))


# ---- layer norm ----
@pytest.mark.parametrize("M,N", [(1, 100), (40, 100), (5, 4096), (600, 300), (37, 999), (3, 20000), (70, 9001)])
def test_layer_norm_gradients_of_rows_far_from_zero(g9, torch_dev, M, N):
    """Means of up to 2^18 times the spread (FP32), whose rounding in stats is 2^-7 of the spread: the gradients are those of the exact
    mean and rstd.

    x - mean is exact where the mean is that large (the two are within a factor of 2); a product and the mean's correction, a sum of
    n = N terms, remain of x̂'s error. A thread sums up to 64 terms and the threads' sums go up a tree, so the forward pass' first
    mean is within 64 units of it, 1; the variance, E(d²) - E(d)² with |E(d)| <= 1 around it, is off by 6 n units and rstd by half."""
    torch = torch_dev
    r = np.random.default_rng(N)
    means = np.resize([2.0 ** 18, -1e5, 7.0 * 2 ** 10, 3.0, 2.0 ** 17 + 0.3], M)[:, None]
    x = (means + r.normal(0, 1, (M, N))).astype(np.float32)
    dy, gamma = r.normal(0, 1, (M, N)).astype(np.float32), (1 + r.normal(0, 0.3, N)).astype(np.float32)
    stats = torch.empty(M, 2, device="cuda")
    g9.layer_norm(gpu(torch, x), gpu(torch, gamma), None, stats=stats)
    x64, dy64 = x.astype(np.float64), dy.astype(np.float64)
    _, mean, rstd = layer_norm(x64, gamma.astype(np.float64), 0.0, 1e-5)
    dx, dg, db = layer_norm_back(dy64, x64, mean, rstd, gamma.astype(np.float64))
    n = N + 8
    er = (3 * n + 4) * U
    xh, gy, rs = np.abs((x64 - mean[:, None]) * rstd[:, None]), np.abs(dy64 * gamma), rstd[:, None]
    off = np.abs(mean[:, None]) * U * rs                     # what the mean's rounding leaves to take off
    exh = 4 * U * (xh + off) + n * U * (xh.mean(1, keepdims=True) + off) + xh * er
    a, c = gy.mean(1, keepdims=True), (gy * (xh + off)).mean(1, keepdims=True)
    q = n * U * c + off * n * U * a + (gy * exh).mean(1, keepdims=True) + exh * a    # the error of mean(g·x̂)
    bound = rs * (n * U * a + xh * q + exh * c + 8 * U * (gy + a + xh * c) + er * (gy + a + xh * c))
    bg, bb = (M + 4) * U * (np.abs(dy64) * xh).sum(0) + (np.abs(dy64) * exh).sum(0), (M + 4) * U * np.abs(dy64).sum(0)
    got = g9.layer_norm_backward(gpu(torch, dy), gpu(torch, x), stats, gpu(torch, gamma))
    near(got[0], dx, bound, np.float32)
    near(got[1], dg, bg, np.float32)
    near(got[2], db, bb, np.float32)
    for grads in ("x", "g", "b", "xb", "gb"):
        some = g9.layer_norm_backward(gpu(torch, dy), gpu(torch, x), stats, gpu(torch, gamma), grads=grads)
        for v, w, key in zip(some, got, "xgb"):
            assert v is None if key not in grads else torch.equal(v, w), (grads, key)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(30000, 40), (7000, 500), (7001, 1001), (2000, 3001), (700, 9001), (600, 16001), (1000, 20001)])
def test_layer_norm_of_many_rows(g9, torch_dev, dtype, M, N):
    """Workgroups with several rows one after the other, in each of the kernels' widths."""
    r = np.random.default_rng(M + N)
    x = (r.normal(0, 1, (M, N)) + r.normal(0, 1, (M, 1))).astype(dtype)
    check_norm(g9, torch_dev, x, (1 + r.normal(0, 0.3, N)).astype(np.float32), r.normal(0, 0.3, N).astype(np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(70, 512), (3, 40000)])
def test_a_refused_capture_leaves_no_kernels(g9, torch_dev, dtype, M, N):
    """A backward norm that is refused in a capture, as its sums need a work buffer, has put nothing into the graph."""
    torch = torch_dev
    t = tensor_type(torch, dtype)
    x = torch.randn(M, N, device="cuda").to(t)
    stats, dX = torch.empty(M, 2, device="cuda"), torch.full((M, N), 5.0, dtype=t, device="cuda")
    g9.layer_norm(x, stats=stats)
    g9.set_nowait(True)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = x + 1
            with pytest.raises(RuntimeError, match="captured"):
                g9.layer_norm_backward(x, x, stats, dX=dX)
        for i in range(3):
            x.mul_(-1)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, x + 1) and (dX == 5).all(), i
    finally:
        g9.set_nowait(False)


# ---- embeddings ----
@pytest.mark.parametrize("T", [262144, 300001])
@pytest.mark.parametrize("V", [500, 70000])
def test_embedding_backward_of_very_many_tokens(g9, torch_dev, T, V):
    """More than 1024 places for a workgroup of the sort, the last of them cut; small integers, whose sums are exact."""
    torch = torch_dev
    r = np.random.default_rng(T)
    ids = r.integers(-3, V + 3, T)
    ids[r.integers(0, T, T // 3)] = V // 2
    dy = r.integers(-1, 2, (T, 5)).astype(np.float16)
    want, _ = embedding_grad(dy, ids, V)
    D, i = gpu(torch, dy), gpu(torch, ids)
    out, buf = laid(torch, np.full((V, 5), 9, np.float32), 3, 1)
    g9.embedding_backward(D, i, V, out=out)
    same(torch, out, want.astype(np.float32))
    g9.embedding_backward(D, i, V, out=out, accumulate=True)
    same(torch, out, 2 * want.astype(np.float32))
    assert untouched(torch, out, buf)
    same(torch, g9.embedding_backward(D.float(), i, V), want.astype(np.float32))
