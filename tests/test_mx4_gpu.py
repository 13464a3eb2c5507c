"""MX4 matrices and products (libgen9blas_llm.so) on a GPU against the definition in 64 bits (tests/mx4_util.py).

Quantised values must equal the definition's bit for bit. Products are held to sum_bound: the products are exact, so only
the FP32 sums and the last rounding differ from the 64-bit result. Covered: both types, lengths from 1 on, row lengths that
end inside a block, a tile and a group of scales, strides and alignments, infinities, NaN, subnormal and huge values, rows
whose scales span the type, and the refusals."""
import ctypes

import numpy as np
import pytest

from mx4_util import packed, quantize, sum_bound, values, zero_block_rows

pytestmark = pytest.mark.gpu


def rng(seed):
    return np.random.default_rng(seed)


def gpu(torch, x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def same(a, b):
    """Equal values, NaN in the same places."""
    return np.array_equal(np.asarray(a, np.float64), np.asarray(b, np.float64), equal_nan=True)


def wide(r, shape, dtype, spread=12.0):
    """Normal values whose size varies over 2^±spread from block to block."""
    x = r.standard_normal(shape) * np.exp2(r.uniform(-spread, spread, (*shape[:-1], 1)))
    return x.astype(dtype)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 31), (3, 32), (16, 128), (17, 129), (5, 512), (33, 515), (16, 4096), (250, 1000), (2, 11008)])
def test_quantize(g9, torch_dev, dtype, rows, K):
    r = rng(rows * 7 + K)
    x = wide(r, (rows, K), dtype, 4.0)
    q = g9.mx4_quantize(gpu(torch_dev, x))
    assert same(g9.mx4_dequantize(q).cpu().numpy(), values(*quantize(x)))


def test_quantize_every_fp16(g9, torch_dev):
    """Every FP16 value beside a largest one of each exponent: all roundings, ties and saturations."""
    every = np.arange(1 << 16, dtype=np.uint16).view(np.float16)
    every = every[np.isfinite(every)]
    for top in (2.0 ** -20, 1.0, 1.75, 6.0, 7.999, 4096.0):
        x = np.zeros((-(-every.size // 31), 32), np.float16)
        x[:, 0] = top
        flat = np.clip(np.resize(every, x.shape[0] * 31), -top, top)
        x[:, 1:] = flat.reshape(-1, 31)
        q = g9.mx4_quantize(gpu(torch_dev, x))
        assert same(g9.mx4_dequantize(q).cpu().numpy(), values(*quantize(x))), top


def test_quantize_special_values(g9, torch_dev):
    x = np.zeros((8, 96), np.float32)
    x[0, 5] = np.inf
    x[1, 40] = np.nan
    x[2, 70] = -np.inf
    x[3, :32] = np.float32(1e-45) * np.arange(32)         # subnormal: the smallest scale
    x[4, :] = np.finfo(np.float32).max
    x[5, 1] = -0.0
    x[6, :32] = np.float32(2.0 ** -126) * np.linspace(0, 4, 32)
    x[7, 32:64] = -np.finfo(np.float32).max
    q = g9.mx4_quantize(gpu(torch_dev, x))
    got = g9.mx4_dequantize(q).cpu().numpy()
    assert same(got, values(*quantize(x)))
    assert np.isnan(got[0, :32]).all() and np.isfinite(got[0, 32:]).all()
    h = np.zeros((2, 64), np.float16)
    h[0, 3], h[1, 33] = np.inf, np.nan
    got = g9.mx4_dequantize(g9.mx4_quantize(gpu(torch_dev, h))).cpu().numpy()
    assert same(got, values(*quantize(h)))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_quantize_strides_stacks_and_reuse(g9, torch_dev, dtype):
    r = rng(3)
    big = gpu(torch_dev, wide(r, (3, 40, 301), dtype, 3.0))
    x = big[:, 1:38, 3:270]                                # rows at any element alignment, strides of rows and matrices
    q = g9.mx4_quantize(x)
    ref = values(*quantize(x.cpu().numpy()))
    assert q.shape == (3, 37, 267) and same(g9.mx4_dequantize(q).cpu().numpy(), ref)
    y = big[:, 2:39, 20:287]
    assert g9.mx4_quantize(y, out=q) is q                  # overwritten whole
    out = torch_dev.full((3, 37, 300), 7.0, device="cuda")
    g9.mx4_dequantize(q, out=out[:, :, 11:278])
    got = out.cpu().numpy()
    assert same(got[:, :, 11:278], values(*quantize(y.cpu().numpy())))
    assert (got[:, :, :11] == 7).all() and (got[:, :, 278:] == 7).all()
    n = x.cpu().numpy()                                    # NumPy in: through the GPU
    assert same(g9.mx4_dequantize(g9.mx4_quantize(n)).cpu().numpy(), ref)


@pytest.mark.parametrize("shape", [(1, 1), (5, 31), (16, 32), (33, 1000), (2, 7, 513), (3, 40, 640)])
def test_load(g9, torch_dev, shape):
    """A checkpoint's codes and scales, any of them: every code, scales 0..255."""
    r = rng(sum(shape))
    codes = r.integers(0, 16, shape).astype(np.uint8)
    scales = r.integers(0, 256, (*shape[:-1], -(-shape[-1] // 32))).astype(np.uint8)
    q = g9.mx4_load(gpu(torch_dev, packed(codes)), gpu(torch_dev, scales), K=shape[-1])
    with np.errstate(over="ignore"):
        want = values(codes, scales).astype(np.float32)
    assert same(g9.mx4_dequantize(q).cpu().numpy(), want)


def check_product(torch, got, a, w, pieces=3):
    a, w = np.asarray(a, np.float64), np.asarray(w, np.float64)
    ref, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    tol = sum_bound(a.shape[1], pieces) * mag
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25
    else:
        tol = tol + 2.0 ** -24 * np.abs(ref)
    err = np.abs(got.cpu().numpy().astype(np.float64) - ref)
    assert np.isfinite(ref).all() and (err <= tol).all(), f"error over the bound by {np.max(err / np.maximum(tol, 1e-300)):.2f}"


SHAPES = [(1, 1, 1), (1, 16, 32), (1, 1000, 4096), (2, 17, 31), (5, 48, 129), (16, 64, 512), (17, 33, 640), (24, 100, 1000), (40, 130, 2051),
          (64, 256, 1024), (65, 300, 513), (100, 257, 4096), (128, 512, 128), (129, 64, 96), (200, 520, 1504), (256, 1024, 2048), (300, 1111, 777), (1000, 96, 352)]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(g9, torch_dev, dtype, M, N, K):
    r = rng(M + N + K)
    a = r.standard_normal((M, K)).astype(dtype)
    codes, scales = quantize(r.standard_normal((N, K)) * np.exp2(r.integers(-9, 2, (N, 1))) / 8)
    W = g9.mx4_load(gpu(torch_dev, packed(codes)), gpu(torch_dev, scales), K=K)
    check_product(torch_dev, g9.mx4_gemm(gpu(torch_dev, a), W), a, values(codes, scales))


@pytest.mark.parametrize("out", [np.float16, np.float32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_quantized(g9, torch_dev, out, M, N, K):
    """Both operands MX4: the products and their scales are exact too."""
    r = rng(M + N + K + 1)
    a = r.standard_normal((M, K)).astype(np.float16)
    codes, scales = quantize(r.standard_normal((N, K)) / 16)
    W = g9.mx4_load(gpu(torch_dev, packed(codes)), gpu(torch_dev, scales), K=K)
    got = g9.mx4_gemm(g9.mx4_quantize(gpu(torch_dev, a)), W, dtype=out)
    assert got.dtype == (torch_dev.float16 if out == np.float16 else torch_dev.float32)
    check_product(torch_dev, got, values(*quantize(a)), values(codes, scales))


def check_large(torch, got, a, w, out):
    """check_product with the 64-bit products on the GPU."""
    ref, mag = a @ w.t(), a.abs() @ w.abs().t()
    tol = sum_bound(a.shape[1]) * mag + (2.0 ** -11 * ref.abs() + 2.0 ** -25 if out == torch.float16 else 2.0 ** -24 * ref.abs())
    assert got.dtype == out and bool(((got.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("K", [96, 200, 384, 512, 640, 1100, 1536])
def test_gemm_quantized_large(g9, torch_dev, K):
    """Enough tiles for one of 256 × 256 a CU, ragged at both ends, for every number of 128-k stages up to a few groups."""
    torch = torch_dev
    g = torch.Generator(device="cuda").manual_seed(K)
    qa = g9.mx4_quantize(torch.randn((4100, K), generator=g, device="cuda"))
    qw = g9.mx4_quantize(torch.randn((4117, K), generator=g, device="cuda") / 8)
    a, w = g9.mx4_dequantize(qa).double(), g9.mx4_dequantize(qw).double()
    for out, t in ((np.float16, torch.float16), (np.float32, torch.float32)):
        check_large(torch, g9.mx4_gemm(qa, qw, dtype=out), a, w, t)


@pytest.mark.parametrize("M,N,K", [(1000, 5000, 256), (513, 4099, 1000), (2050, 2050, 640)])
def test_gemm_large(g9, torch_dev, M, N, K):
    """More tiles than CUs: k is not split."""
    torch = torch_dev
    g = torch.Generator(device="cuda").manual_seed(M)
    W = g9.mx4_quantize(torch.randn((N, K), generator=g, device="cuda") / 8)
    w = g9.mx4_dequantize(W).double()
    for t in (torch.float16, torch.float32):
        a = torch.randn((M, K), generator=g, device="cuda").to(t)
        check_large(torch, g9.mx4_gemm(a, W), a.double(), w, t)


@pytest.mark.parametrize("M,N,K", [(16, 8192, 4096), (16, 2048, 8192), (9, 2050, 8200), (1, 16400, 200), (5, 17003, 129), (16, 22016, 96)])
def test_gemm_few_rows_large(g9, torch_dev, M, N, K):
    """Up to 16 rows of products that read much, or whose columns fill the GPU without a split of k: 128 columns a workgroup."""
    torch = torch_dev
    g = torch.Generator(device="cuda").manual_seed(N)
    W = g9.mx4_quantize(torch.randn((N, K), generator=g, device="cuda") / 8)
    w = g9.mx4_dequantize(W).double()
    for t in (torch.float16, torch.float32):
        big = torch.randn((M, K + 3), generator=g, device="cuda").to(t)
        for a in (big[:, :K], big[:, 1:K + 1]):
            out = torch.full((M, N + 5), 3.0, dtype=t, device="cuda")
            g9.mx4_gemm(a, W, C=out[:, 2:N + 2])
            check_large(torch, out[:, 2:N + 2], a.double(), w, t)
            assert bool((out[:, :2] == 3.0).all()) and bool((out[:, N + 2:] == 3.0).all())


@pytest.mark.parametrize("K", [96, 200, 384, 512, 640, 1100, 1536])
def test_gemm_quantized_middle(g9, torch_dev, K):
    """More tiles of 16 × 16 than eight a CU, too few of 256 × 256."""
    torch = torch_dev
    g = torch.Generator(device="cuda").manual_seed(K)
    qa = g9.mx4_quantize(torch.randn((700, K), generator=g, device="cuda"))
    qw = g9.mx4_quantize(torch.randn((1301, K), generator=g, device="cuda") / 8)
    a, w = g9.mx4_dequantize(qa).double(), g9.mx4_dequantize(qw).double()
    for out, t in ((np.float16, torch.float16), (np.float32, torch.float32)):
        check_large(torch, g9.mx4_gemm(qa, qw, dtype=out), a, w, t)


@pytest.mark.parametrize("M,N", [(4100, 4117), (700, 1301)])
@pytest.mark.parametrize("K", [768, 870, 1280, 1400])
def test_gemm_quantized_stages_after_whole_groups(g9, torch_dev, M, N, K):
    """Six, seven, ten and eleven 128-k stages: two and three of them after the last whole group of four, in both tilings."""
    torch = torch_dev
    g = torch.Generator(device="cuda").manual_seed(K + M)
    qa = g9.mx4_quantize(torch.randn((M, K), generator=g, device="cuda"))
    qw = g9.mx4_quantize(torch.randn((N, K), generator=g, device="cuda") / 8)
    a, w = g9.mx4_dequantize(qa).double(), g9.mx4_dequantize(qw).double()
    for out, t in ((np.float16, torch.float16), (np.float32, torch.float32)):
        check_large(torch, g9.mx4_gemm(qa, qw, dtype=out), a, w, t)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("M,N,K", [(300, 5000, 200), (700, 4099, 129), (1100, 4099, 645)])
def test_gemm_large_strides_and_nan(g9, torch_dev, dtype, M, N, K):
    """Tiles of 64 rows by 128 and 256 columns: A at any alignment, nothing written beside C, an infinity or NaN stays in its row."""
    torch = torch_dev
    t = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(M)
    W = g9.mx4_quantize(torch.randn((N, K), generator=g, device="cuda") / 8)
    w = g9.mx4_dequantize(W).double()
    big = torch.randn((M, K + 5), generator=g, device="cuda").to(t)
    for off in (0, 1, 2):
        a = big[:, off:off + K]
        out = torch.full((M + 2, N + 7), 3.0, dtype=t, device="cuda")
        g9.mx4_gemm(a, W, C=out[1:M + 1, 2:N + 2])
        check_large(torch, out[1:M + 1, 2:N + 2], a.double(), w, t)
        out[1:M + 1, 2:N + 2] = 3.0
        assert bool((out == 3.0).all())
    a = big[:, :K].clone()
    a[5, 7], a[M - 2, K - 1] = float("nan"), float("inf")
    rest = [i for i in range(M) if i not in (5, M - 2)]
    got = g9.mx4_gemm(a, W)
    check_large(torch, got[rest], a[rest].double(), w, t)
    assert bool(got[5].isnan().all()) and not bool(got[M - 2].isfinite().any())


@pytest.mark.parametrize("step", [256, 260, 262, 263])
def test_gemm_large_rows_in_place(g9, torch_dev, step):
    """Whole 128-k chunks of FP16 rows for the tile kernel, which copies them to LDS from where they lie if all rows begin at multiples of
    four bytes, of any sixteen; from odd elements, and at odd strides, by way of the work space."""
    torch = torch_dev
    M, N, K = 1000, 4400, 256
    g = torch.Generator(device="cuda").manual_seed(step)
    W = g9.mx4_quantize(torch.randn((N, K), generator=g, device="cuda") / 8)
    w = g9.mx4_dequantize(W).double()
    flat = torch.randn(M * step + 8, generator=g, device="cuda").half()
    for off in (0, 1, 2, 4, 6):
        a = flat.as_strided((M, K), (step, 1), off)
        check_large(torch, g9.mx4_gemm(a, W), a.double(), w, torch.float16)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("M", [1, 7, 33, 90, 260])
def test_gemm_strides(g9, torch_dev, dtype, M):
    """A at any alignment and row stride; C with a row stride, nothing written beside it."""
    r = rng(M)
    N, K = 200, 645
    big = gpu(torch_dev, r.standard_normal((M + 1, K + 9)).astype(dtype))
    codes, scales = quantize(r.standard_normal((N, K)) / 8)
    W = g9.mx4_load(gpu(torch_dev, packed(codes)), gpu(torch_dev, scales), K=K)
    for off in (0, 1, 3):
        a = big[1:, off:off + K]
        out = torch_dev.full((M + 2, N + 7), 3.0, dtype=a.dtype, device="cuda")
        g9.mx4_gemm(a, W, C=out[1:M + 1, 2:N + 2])
        check_product(torch_dev, out[1:M + 1, 2:N + 2], a.cpu().numpy(), values(codes, scales))
        out[1:M + 1, 2:N + 2] = 3.0
        assert bool((out == 3.0).all())
    q = g9.mx4_quantize(big[1:, 2:2 + K])
    out = torch_dev.full((M, N + 5), 3.0, dtype=torch_dev.float32, device="cuda")
    g9.mx4_gemm(q, W, C=out[:, 1:N + 1])
    check_product(torch_dev, out[:, 1:N + 1], values(*quantize(big[1:, 2:2 + K].cpu().numpy())), values(codes, scales))
    assert bool((out[:, 0] == 3.0).all()) and bool((out[:, N + 1:] == 3.0).all())


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_inputs_of_any_layout(g9, torch_dev, dtype):
    """Layouts that the C entry points do not take are copied: repeated and overlapping rows, permuted dimensions, NumPy's negative
    strides."""
    torch = torch_dev
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((6, 5, 96), generator=g, device="cuda").to(getattr(torch, dtype))
    flat = x.reshape(-1)
    W = g9.mx4_quantize(torch.randn((40, 96), generator=g, device="cuda"))
    for a in (x[0, :1].expand(9, 96), flat.as_strided((9, 96), (7, 1)), x[:, 0], x[0, :, :48].expand(2, 5, 48).reshape(5, 96), x[0].t().contiguous().t()):
        assert bool((g9.mx4_gemm(a, W) == g9.mx4_gemm(a.contiguous(), W)).all())
        assert bool((g9.mx4_dequantize(g9.mx4_quantize(a)) == g9.mx4_dequantize(g9.mx4_quantize(a.contiguous()))).all())
    for a in (x.transpose(0, 1), x[:1].expand(3, 5, 96), x[:, :1].expand(6, 4, 96), flat.as_strided((3, 5, 40), (11, 2, 1)), x.transpose(1, 2)):
        assert bool((g9.mx4_dequantize(g9.mx4_quantize(a)) == g9.mx4_dequantize(g9.mx4_quantize(a.contiguous()))).all())
    n = x[0].cpu().numpy()
    for a in (n[::-1], n[:, ::-1], n[::2], n.T[::-1].T):
        assert np.array_equal(g9.mx4_gemm(a, W), g9.mx4_gemm(a.copy(), W))
    c, s = np.arange(4 * 48, dtype=np.uint8).reshape(4, 48), np.arange(120, 132, dtype=np.uint8).reshape(4, 3)
    assert same(g9.mx4_dequantize(g9.mx4_load(c[::-1], s[::-1])).cpu(), g9.mx4_dequantize(g9.mx4_load(c[::-1].copy(), s[::-1].copy())).cpu())


def test_row_strides_past_32_bits(g9, torch_roomy):
    """The C entry points have row strides of 31 bits: inputs of longer ones are copied, such results are refused."""
    torch = torch_roomy
    far = (1 << 32) + 64
    buf = torch.zeros(far + 64, dtype=torch.float16, device="cuda")
    a = buf.as_strided((2, 64), (far, 1))
    buf[:128] = torch.arange(128, device="cuda") / 16
    a[1] = 1.0
    W = g9.mx4_quantize(torch.ones((64, 64), device="cuda"))
    assert bool((g9.mx4_gemm(a, W) == g9.mx4_gemm(a.contiguous(), W)).all())
    assert bool((g9.mx4_dequantize(g9.mx4_quantize(a)) == g9.mx4_dequantize(g9.mx4_quantize(a.contiguous()))).all())
    got, want = g9.moe_route(a, 2), g9.moe_route(a.contiguous(), 2)
    assert bool((got[0] == want[0]).all()) and bool((got[1] == want[1]).all())
    with pytest.raises(ValueError):
        g9.mx4_gemm(a.contiguous(), W, C=a)
    stack = g9.mx4_quantize(torch.ones((2, 64, 64), device="cuda"))    # strides of tokens are of 64 bits
    ids = torch.ones((2, 1), dtype=torch.int32, device="cuda")
    y = g9.moe_gemm(a, ids, stack)
    assert bool((y == g9.moe_gemm(a.contiguous(), ids, stack)).all())
    g9.moe_gemm(a.contiguous(), ids, stack, C=buf.as_strided((2, 1, 64), (far, 64, 1)))
    assert bool((a == y[:, 0]).all()) and bool((buf[64:128] == torch.arange(64, 128, device="cuda") / 16).all())


def test_rows_of_two_billion(g9, torch_roomy):
    """The longest rows that a matrix has; longer ones are refused."""
    torch = torch_roomy
    K = (1 << 31) - 128
    L = g9._llm_library()
    for k in (K + 1, K + 127):
        assert L.gen9blas_mx4_create(1, 1, k) is None and L.gen9blas_llm_last_status() == -2
    x = torch.zeros((1, K), dtype=torch.float16, device="cuda")
    at, v = torch.tensor([0, 12345, K // 2 + 1, K - 1], device="cuda"), torch.tensor([2.0, -1.0, 0.5, 3.0], device="cuda")
    x[0, at] = v.half()
    q = g9.mx4_quantize(x)
    d = g9.mx4_dequantize(q)
    assert bool((d[0, at] == v).all()) and int(torch.count_nonzero(d)) == 4
    del d
    assert float(g9.mx4_gemm(x, q)) == float((v * v).sum())
    del x, q
    for shape in ((1, (1 << 32) + 5), ((1 << 32) + 1, 4), ((1 << 32) + 1, 2, 2)):    # not cut to their low 32 bits
        with pytest.raises(ValueError):
            g9.MX4(*shape)
    tall = torch.empty(((1 << 31) + 1, 1), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        g9.mx4_gemm(tall, g9.MX4(4, 1))
    with pytest.raises(ValueError):
        g9.moe_route(tall, 1)


def test_dtype_that_contradicts_is_refused(g9, torch_dev):
    """dtype chooses the result's type of two MX4 operands; where it is given already, another dtype is not ignored."""
    torch = torch_dev
    a = torch.ones((4, 64), dtype=torch.float16, device="cuda")
    W = g9.mx4_quantize(torch.ones((8, 64), device="cuda"))
    q = g9.mx4_quantize(a)
    assert g9.mx4_gemm(a, W, dtype=np.float16).dtype == torch.float16
    C = torch.empty((4, 8), device="cuda")
    assert g9.mx4_gemm(q, W, C=C, dtype=np.float32) is C
    with pytest.raises(TypeError):
        g9.mx4_gemm(a, W, dtype=np.float32)
    with pytest.raises(TypeError):
        g9.mx4_gemm(q, W, C=C, dtype=np.float16)


@pytest.mark.parametrize("M", [1, 16, 40, 70, 130, 300])
def test_gemm_fp32_is_fp32(g9, torch_dev, M):
    """FP32 activations keep their 24 bits: over 32 products of one sign the relative error is a few units of 2^-24, where
    activations cut to 16 bits would be 2^-17 off."""
    r = rng(M)
    N, K = 64, 32
    a = r.uniform(1, 2, (M, K)).astype(np.float32)
    codes = r.integers(1, 8, (N, K)).astype(np.uint8)
    scales = r.integers(100, 150, (N, 1)).astype(np.uint8)
    W = g9.mx4_load(gpu(torch_dev, packed(codes)), gpu(torch_dev, scales), K=K)
    got = g9.mx4_gemm(gpu(torch_dev, a), W).cpu().numpy().astype(np.float64)
    ref = a.astype(np.float64) @ values(codes, scales).T
    assert np.max(np.abs(got - ref) / ref) <= 16 * 2.0 ** -24


@pytest.mark.parametrize("M", [1, 20, 100, 300])
def test_gemm_scales_of_any_size(g9, torch_dev, M):
    """Scales far from one: FP32 takes any within FP32's range; FP16 activations take rows of any scale whose blocks lie
    within 2^36 of the row's largest, blocks of zeros with any scale beside them."""
    r = rng(M)
    N, K = 48, 1024
    codes = r.integers(0, 16, (N, K)).astype(np.uint8)
    scales = (r.integers(20, 200, (N, 1)) + r.integers(0, 17, (N, K // 32))).astype(np.uint8)
    W = g9.mx4_load(gpu(torch_dev, packed(codes)), gpu(torch_dev, scales), K=K)
    a = r.standard_normal((M, K)).astype(np.float32)
    check_product(torch_dev, g9.mx4_gemm(gpu(torch_dev, a), W), a, values(codes, scales))
    base = r.integers(110, 135, (N, 1))
    scales = (base - r.integers(0, 37, (N, K // 32))).astype(np.uint8)
    scales[:, 3] = 250
    codes[:, 96:128] = 8 * r.integers(0, 2, (N, 32))       # zeros of both signs under a large scale
    W = g9.mx4_load(gpu(torch_dev, packed(codes)), gpu(torch_dev, scales), K=K)
    h = (r.standard_normal((M, K)) / 256).astype(np.float16)
    ref = values(codes, scales)
    assert np.abs(h.astype(np.float64) @ ref.T).max() < 6e4
    check_product(torch_dev, g9.mx4_gemm(gpu(torch_dev, h), W), h, ref)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("M", [1, 20, 100, 500, 1000])
def test_gemm_blocks_of_zeros_with_any_scale(g9, torch_dev, dtype, M):
    """A block of zeros is zeros whatever its scale says, in rows of any largest scale and in rows of nothing but zeros; a NaN block
    (scale 255) stays NaN. Rows enough for every kernel that takes these M. A in steps of 2^-10, so that no sum of FP32 is rounded, the
    subnormal ones of the least scales among them."""
    torch = torch_dev
    r = rng(M)
    parts = [zero_block_rows(r, 640) for _ in range(4)]
    codes, scales = (np.concatenate([p[i] for p in parts]) for i in (0, 1))
    nan = (scales == 255).any(1)
    W = g9.mx4_load(gpu(torch, packed(codes)), gpu(torch, scales), K=640)
    a = gpu(torch, (r.integers(-64, 65, (M, 640)) / 1024).astype(dtype))
    got = g9.mx4_gemm(a, W)
    assert bool(got[:, gpu(torch, nan)].isnan().all())
    assert bool(got[:, gpu(torch, ~nan)].isfinite().all())
    check_large(torch, got[:, gpu(torch, ~nan)], a.double(), gpu(torch, values(codes[~nan], scales[~nan])), got.dtype)


@pytest.mark.parametrize("M", [1, 20, 100, 500, 1000])
def test_gemm_quantized_nan_block_stays_nan(g9, torch_dev, M):
    """The codes of a NaN block are zeros: a block of zeros must not be taken for it, nor it for one."""
    torch = torch_dev
    w = torch.zeros((4500, 640), device="cuda")
    w[7, 100], w[4499, 639], w[300, 40] = float("nan"), float("inf"), 1.0
    got = g9.mx4_gemm(torch.ones((M, 640), dtype=torch.float16, device="cuda"), g9.mx4_quantize(w))
    want = torch.zeros((M, 4500), dtype=torch.float16, device="cuda")
    want[:, 7], want[:, 4499], want[:, 300] = float("nan"), float("nan"), 1.0
    assert same(got.cpu().numpy(), want.cpu().numpy())


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("M", [3, 50, 140, 300])
def test_gemm_infinities_and_nan(g9, torch_dev, dtype, M):
    """An infinity or NaN in a row of A, or a NaN block of W, reaches its own row or column and nothing else; the type's
    largest values stay finite where their products are."""
    r = rng(M)
    N, K = 40, 300
    a = r.standard_normal((M, K)).astype(dtype)
    a[0, 7], a[1, 299] = np.inf, np.nan
    if dtype == np.float32:
        a[1, 299] = np.array([0x7f800001], np.uint32).view(np.float32)[0]   # a NaN whose payload is its lowest bit
    a[2, :] = 0
    a[2, 5] = -np.finfo(dtype).max
    codes = r.integers(1, 8, (N, K)).astype(np.uint8)
    codes[:, 5] = 1                                       # 0.5
    scales = np.full((N, 10), 125, np.uint8)
    scales[11, 4] = 255
    W = g9.mx4_load(gpu(torch_dev, packed(codes)), gpu(torch_dev, scales), K=K)
    got = g9.mx4_gemm(gpu(torch_dev, a), W).cpu().numpy().astype(np.float64)
    assert np.isnan(got[:, 11]).all()
    got, w = np.delete(got, 11, 1), np.delete(values(codes, scales), 11, 0)
    assert (got[0] == np.inf).all() and np.isnan(got[1]).all()
    assert (got[2] == -float(np.finfo(dtype).max) / 8).all()
    check_product(torch_dev, torch_dev.from_numpy(got[3:].astype(dtype)), a[3:], w)


def test_gemm_quantized_nan(g9, torch_dev):
    r = rng(5)
    a = r.standard_normal((70, 256)).astype(np.float32)
    a[4, 100] = np.inf
    wv = r.standard_normal((50, 256)).astype(np.float32)
    wv[9, 0] = np.nan
    got = g9.mx4_gemm(g9.mx4_quantize(gpu(torch_dev, a)), g9.mx4_quantize(gpu(torch_dev, wv)), dtype=np.float32).cpu().numpy()
    want = np.zeros((70, 50), bool)
    want[4], want[:, 9] = True, True
    assert np.array_equal(np.isnan(got), want) and np.isfinite(got[~want]).all()


def test_gemm_is_repeatable(g9, torch_dev):
    r = rng(8)
    for M, N, K in ((1, 4096, 4096), (24, 1000, 11008), (300, 512, 4096)):
        for dtype in (np.float16, np.float32):
            a = gpu(torch_dev, r.standard_normal((M, K)).astype(dtype))
            W = g9.mx4_quantize(gpu(torch_dev, r.standard_normal((N, K)).astype(np.float32)))
            first = g9.mx4_gemm(a, W)
            assert all(bool((g9.mx4_gemm(a, W) == first).all()) for _ in range(3))


def test_nowait_and_streams(g9, torch_dev):
    """Queued calls in a row, and tensors made and read on a torch stream of their own, without any wait by the caller."""
    torch = torch_dev
    r = rng(4)
    W = g9.mx4_quantize(gpu(torch, r.standard_normal((512, 512)).astype(np.float32)))
    a = r.standard_normal((64, 512)).astype(np.float32)
    ref = g9.mx4_gemm(gpu(torch, a), W).cpu().numpy()
    g9.set_nowait(True)
    try:
        side = torch.cuda.Stream()
        for _ in range(20):
            with torch.cuda.stream(side):
                x = torch.from_numpy(a).cuda(non_blocking=True)
                x = (x * 2).contiguous() / 2
                y = g9.mx4_gemm(x, W) * 1.0
            side.synchronize()
            assert np.array_equal(y.cpu().numpy(), ref)
        y = g9.mx4_gemm(torch.from_numpy(a).cuda(), W)
        assert np.array_equal((y + 0).cpu().numpy(), ref)
    finally:
        g9.set_nowait(False)
        g9.flush()


def test_refusals(g9, torch_dev):
    torch = torch_dev
    L = g9._llm_library()
    x = torch.ones((4, 64), device="cuda")
    W = g9.mx4_quantize(torch.ones((8, 64), device="cuda"))
    C = torch.full((4, 8), 5.0, device="cuda")
    host = np.ones((4, 64), np.float32)
    INVALID, UNSUPPORTED = -3, -2
    assert L.gen9blas_mx4_gemm(3, 4, x.data_ptr(), 64, W._handle, C.data_ptr(), 8) == UNSUPPORTED
    assert L.gen9blas_mx4_gemm(1, 4, x.data_ptr(), 63, W._handle, C.data_ptr(), 8) == INVALID
    assert L.gen9blas_mx4_gemm(1, 4, x.data_ptr(), 64, W._handle, C.data_ptr(), 7) == INVALID
    assert L.gen9blas_mx4_gemm(1, 4, host.ctypes.data, 64, W._handle, C.data_ptr(), 8) == INVALID
    assert b"A" in L.gen9blas_llm_error() and L.gen9blas_llm_last_status() == INVALID
    assert L.gen9blas_mx4_gemm(1, 4, None, 64, W._handle, C.data_ptr(), 8) == INVALID
    assert L.gen9blas_mx4_gemm(1, 4, x.data_ptr(), 64, None, C.data_ptr(), 8) == INVALID
    assert L.gen9blas_mx4_gemm(1, 0, None, 64, W._handle, None, 8) == 0
    assert L.gen9blas_mx4_gemm_q(1, W._handle, None, C.data_ptr(), 8) == INVALID
    assert L.gen9blas_mx4_quantize(0, x.data_ptr(), 10, 0, W._handle) == INVALID
    assert L.gen9blas_mx4_create(1, 0, 4) is None and L.gen9blas_llm_last_status() == INVALID
    L.gen9blas_mx4_free(None)
    torch.cuda.synchronize()
    assert bool((C == 5.0).all())
    stack = g9.mx4_quantize(torch.ones((2, 8, 64), device="cuda"))
    with pytest.raises(ValueError):
        g9.mx4_gemm(x, stack)
    with pytest.raises(ValueError):
        g9.mx4_gemm(torch.ones((4, 65), device="cuda"), W)
    with pytest.raises(ValueError):
        g9.mx4_gemm(x, W, C=torch.empty((4, 9), device="cuda"))
    with pytest.raises(ValueError):
        g9.mx4_gemm(x, W, C=torch.empty((4, 8), dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError):
        g9.mx4_quantize(x, out=W)
    with pytest.raises(ValueError):
        g9.mx4_load(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8))
    with pytest.raises(TypeError):
        g9.mx4_load(torch.zeros((4, 16)), torch.zeros((4, 1), dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        g9.MX4(0, 5)
    # NumPy operands give NumPy results
    y = g9.mx4_gemm(host, W)
    assert isinstance(y, np.ndarray) and (y == 64).all()
