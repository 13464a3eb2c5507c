"""Mixture of experts (libgen9blas_llm.so) on a GPU: the router and the experts' products, against 64-bit NumPy.

The router's choices are compared exactly where equal choices decide (logits on a coarse grid, the lowest index first), and
for random logits against the 64-bit choices: an expert may stand in for another only where their choices are within the
rounding of an FP32 score (2^-20). Products have the bounds of tests/mx4_util.py; the gate's SiLU passes on the error of its
argument with a slope of at most 1.1, and adds a few units of 2^-23 of its own."""
import numpy as np
import pytest

from mx4_util import packed, quantize, sum_bound, values, zero_block_rows

pytestmark = pytest.mark.gpu


def gpu(torch, x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def route64(x, k, bias, score, groups, top_groups, renorm, scale):
    """ids, weights and all scores and choices in 64 bits; masked experts are -inf in the choices."""
    x = np.asarray(x, np.float64)
    T, E = x.shape
    if score == "sigmoid":
        s = 1 / (1 + np.exp(-x))
        choice = np.where(x > -np.inf, s, -np.inf)
    else:
        m = x.max(1, keepdims=True)
        with np.errstate(invalid="ignore"):
            p = np.where(x > -np.inf, np.exp(x - m), 0)
            s = p / np.maximum(p.sum(1, keepdims=True), 1e-300)
        choice = np.where(x > -np.inf, s if bias is not None else x, -np.inf)
    if bias is not None:
        choice = choice + bias
    if groups > 1:
        per = np.sort(choice.reshape(T, groups, -1), -1)[..., ::-1]
        of = per[..., 0].copy()
        if score == "sigmoid" and per.shape[-1] > 1:
            of += np.where(per[..., 1] > -np.inf, per[..., 1], 0)
        order = np.argsort(-of, axis=1, kind="stable")
        keep = np.zeros((T, groups), bool)
        np.put_along_axis(keep, order[:, :top_groups], True, 1)
        choice = np.where(np.repeat(keep, E // groups, 1), choice, -np.inf)
    ids = np.argsort(-choice, axis=1, kind="stable")[:, :k]
    left = np.take_along_axis(choice, ids, 1) > -np.inf
    w = np.where(left, np.take_along_axis(s, ids, 1), 0)
    ids = np.where(left, ids, -1)
    if renorm:
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return ids, w * scale, s, choice


def check_route(g9, torch, x, k, bias=None, score="softmax", groups=1, top_groups=1, renorm=True, scale=1.0):
    """Where the 64-bit groups and experts are decided by more than FP32's rounding, ids must agree; all weights must be
    those of the chosen experts."""
    ids, w = g9.moe_route(gpu(torch, x), k, bias=None if bias is None else gpu(torch, bias), score=score, groups=groups,
                          top_groups=top_groups, renorm=renorm, scale=scale)
    ids, w = ids.cpu().numpy(), w.cpu().numpy()
    want, want_w, s, choice = route64(x, k, bias, score, groups, top_groups, renorm, scale)
    differ = (ids != want).any(1)
    for t in np.nonzero(differ)[0]:
        # another expert, or another order: only between choices that are as good as equal
        a, b = choice[t][ids[t]], choice[t][want[t]]
        assert (np.abs(a - b) <= 2.0 ** -20).all() and len(set(ids[t])) == k, (t, ids[t], want[t])
    assert differ.mean() <= 0.01
    same = ~differ
    assert np.allclose(w[same], want_w[same], rtol=64 * 2.0 ** -24, atol=1e-30)
    return ids, w


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (3, 7, 7), (5, 64, 64), (100, 65, 6), (17, 128, 4), (250, 256, 8), (33, 384, 10), (9, 512, 2), (7, 1000, 33), (4, 1024, 64)])
def test_route(g9, torch_dev, dtype, score, T, E, k):
    r = np.random.default_rng(T + E + k)
    # distinct logits in each row (a shuffled grid), so that FP16 has no ties
    x = (np.argsort(r.random((T, E)), 1) / E * 6 - 3).astype(dtype)
    for renorm, scale in ((True, 1.0), (False, 2.5)):
        check_route(g9, torch_dev, x, k, None, score, renorm=renorm, scale=scale)
    bias = r.normal(0, 0.1, E).astype(np.float32)
    check_route(g9, torch_dev, x.astype(np.float32), k, bias, score)


@pytest.mark.parametrize("score,bias", [("softmax", False), ("sigmoid", False), ("sigmoid", True), ("softmax", True)])
@pytest.mark.parametrize("E,groups,top,k", [(64, 8, 4, 8), (256, 8, 4, 8), (40, 4, 1, 10), (96, 3, 2, 6), (160, 8, 7, 5), (64, 64, 9, 9), (64, 32, 5, 3), (1024, 16, 2, 20)])
def test_route_groups(g9, torch_dev, score, bias, E, groups, top, k):
    r = np.random.default_rng(E + groups)
    x = r.normal(0, 1.5, (300, E)).astype(np.float32)
    b = r.normal(0, 0.1, E).astype(np.float32) if bias else None
    check_route(g9, torch_dev, x, k, b, score, groups, top)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lowest_index(g9, torch_dev, dtype, score):
    r = np.random.default_rng(2)
    x = r.integers(-1, 2, (200, 96)).astype(dtype)
    x[5] = 0
    x[6, ::2] = -0.0
    x[6, 1::2] = 0.0
    for groups, top in ((1, 1), (8, 3)):
        ids, _ = g9.moe_route(gpu(torch_dev, x), 12, score=score, groups=groups, top_groups=top)
        assert np.array_equal(ids.cpu().numpy(), route64(x, 12, None, score, groups, top, True, 1.0)[0])


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_masks(g9, torch_dev, dtype, score):
    """Experts masked by -inf, rows that leave fewer than k or none, the type's lowest value, infinities and NaN."""
    r = np.random.default_rng(3)
    x = (np.argsort(r.random((12, 64)), 1) / 16 - 2).astype(dtype)
    x[0, :] = -np.inf                       # nothing left
    x[1, 3:] = -np.inf                      # three left
    x[2, ::2] = -np.inf
    x[3, :] = np.finfo(dtype).min           # all alike, and as low as the type goes
    x[4, 10:] = np.finfo(dtype).min
    x[5, 7] = np.nan
    with np.errstate(over="ignore"):
        ids, w = check_route(g9, torch_dev, np.delete(x, (3, 5), 0), 8, None, score)
    assert (ids[0] == -1).all() and (w[0] == 0).all()
    assert sorted(ids[1][:3]) == [0, 1, 2] and (ids[1][3:] == -1).all() and (w[1][3:] == 0).all() and abs(w[1].sum() - 1) < 1e-6
    ids, w = (v.cpu().numpy() for v in g9.moe_route(gpu(torch_dev, x), 8, score=score))
    assert np.array_equal(ids[3], np.arange(8))
    assert np.allclose(w[3], 1 / 8 if score == "softmax" else 0)     # sigmoids of 0: nothing to share out
    assert np.isnan(w[5]).all() and 7 not in ids[5]
    # groups that are masked whole or but for one expert
    x = (np.argsort(r.random((4, 64)), 1) / 16 - 2).astype(np.float32)
    x[0, 8:] = -np.inf
    x[1, :56] = -np.inf
    x[2, :] = -np.inf
    x[3, 1:32] = -np.inf
    ids, w = check_route(g9, torch_dev, x, 6, None, score, 8, 2)
    assert (ids[2] == -1).all() and (ids[0] < 8).all()
    # an infinite logit of a sigmoid is a score of 1
    x = np.zeros((1, 8), np.float32)
    x[0, 5] = np.inf
    ids, w = (v.cpu().numpy() for v in g9.moe_route(gpu(torch_dev, x), 2, score="sigmoid", renorm=False))
    assert list(ids[0]) == [5, 0] and list(w[0]) == [1.0, 0.5]


def test_route_strides_and_out(g9, torch_dev):
    torch = torch_dev
    r = np.random.default_rng(5)
    big = r.normal(size=(50, 101)).astype(np.float16)
    x = gpu(torch, big)[3:40, 5:95]
    ids, w = torch.empty((37, 4), dtype=torch.int32, device="cuda"), torch.empty((37, 4), device="cuda")
    got = g9.moe_route(x, 4, out=(ids, w))
    assert got[0] is ids and got[1] is w
    want = g9.moe_route(x.contiguous(), 4)
    assert bool((ids == want[0]).all()) and bool((w == want[1]).all())
    n = g9.moe_route(big[3:40, 5:95], 4)
    assert isinstance(n[0], np.ndarray) and np.array_equal(n[0], ids.cpu().numpy())
    e = g9.moe_route(torch.empty((0, 8), device="cuda"), 2)
    assert e[0].shape == (0, 2)


def weights(r, torch, g9, E, N, K):
    codes, scales = quantize(r.standard_normal((E, N, K)) * np.exp2(r.integers(-6, 1, (E, N, 1))) / 8)
    return g9.mx4_load(gpu(torch, packed(codes)), gpu(torch, scales), K=K), values(codes, scales)


def experts64(x, ids, w, gate=None, weights=None, sums=None):
    """The result and its error bound before the last rounding. `sums`: the bound of a sum over its magnitudes."""
    T, S = ids.shape
    E, N, K = w.shape
    x = np.asarray(x, np.float64)
    x = np.broadcast_to(x[:, None], (T, S, K)) if x.ndim == 2 else x
    y, dy = np.zeros((T, S, N)), np.zeros((T, S, N))
    b = sum_bound(K)
    for e in range(E):
        t, s = np.nonzero(ids == e)
        if not len(t):
            continue
        rows = x[t, s]
        u, du = rows @ w[e].T, b * (np.abs(rows) @ np.abs(w[e]).T)
        if gate is not None:
            z, dz = rows @ gate[e].T, b * (np.abs(rows) @ np.abs(gate[e]).T)
            a = z / (1 + np.exp(-z))
            u, du = a * u, 1.1 * dz * (np.abs(u) + du) + np.abs(a) * du + 16 * 2.0 ** -23 * np.abs(a * u)
        y[t, s], dy[t, s] = u, du
    if weights is None:
        return y, dy
    g = np.asarray(weights, np.float64)[..., None] * (ids >= 0)[..., None] * (ids < E)[..., None]
    out = (g * y).sum(1)
    return out, (np.abs(g) * (dy + (S + 1) * 2.0 ** -23 * np.abs(y))).sum(1)


def check_experts(torch, got, ref, tol):
    tol = tol + (2.0 ** -11 * np.abs(ref) + 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -23 * np.abs(ref))
    err = np.abs(got.cpu().numpy().astype(np.float64) - ref)
    assert (err <= tol).all(), f"error over the bound by {np.max(err / np.maximum(tol, 1e-300)):.2f}"


CASES = [(1, 1, 1, 16, 32), (1, 8, 16, 64, 512), (2, 3, 5, 33, 131), (7, 2, 4, 48, 640), (24, 4, 64, 130, 200), (65, 1, 3, 100, 96), (100, 6, 8, 64, 513), (300, 2, 4, 257, 256), (513, 4, 9, 96, 160)]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("T,S,E,N,K", CASES)
def test_experts(g9, torch_dev, dtype, T, S, E, N, K):
    """Every form: one row a token or one a place, gated or not, joined or not; some places empty."""
    r = np.random.default_rng(T + S + E + N + K)
    ids = np.argsort(r.random((T, E)), 1)[:, :S].astype(np.int32)
    if T > 1:
        ids[r.random(ids.shape) < 0.1] = -1
        ids[0, 0] = E + 3                   # no expert either
    W, w = weights(r, torch_dev, g9, E, N, K)
    G, g = weights(r, torch_dev, g9, E, N, K)
    share = r.random((T, S)).astype(np.float32)
    if T > 1:
        share[ids < 0] = np.nan             # weights of empty places are not read
    i = gpu(torch_dev, ids)
    for x in (r.standard_normal((T, K)), r.standard_normal((T, S, K))):
        x = x.astype(dtype)
        xd = gpu(torch_dev, x)
        for gate in (False, True):
            for join in (False, True):
                got = g9.moe_gemm(xd, i, W, gate=G if gate else None, weights=gpu(torch_dev, share) if join else None)
                ref, tol = experts64(x, ids, w, g if gate else None, np.nan_to_num(share) if join else None)
                check_experts(torch_dev, got, ref, tol)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("T,S,E,N,K", [(30, 2, 4, 100, 300), (150, 4, 64, 2070, 160), (16, 4, 9, 300, 260)])
def test_experts_of_seven_places_and_more(g9, torch_dev, dtype, T, S, E, N, K):
    """Tiles of 32 rows (FP16), without a plan and with one; enough experts and columns for 256 columns a workgroup."""
    r = np.random.default_rng(T + N)
    ids = np.argsort(r.random((T, E)), 1)[:, :S].astype(np.int32)
    ids[r.random(ids.shape) < 0.1] = -1
    W, w = weights(r, torch_dev, g9, E, N, K)
    G, g = weights(r, torch_dev, g9, E, N, K)
    share = r.random((T, S)).astype(np.float32)
    x = r.standard_normal((T, S, K)).astype(dtype)
    for gate in (False, True):
        for join in (False, True):
            got = g9.moe_gemm(gpu(torch_dev, x), gpu(torch_dev, ids), W, gate=G if gate else None, weights=gpu(torch_dev, share) if join else None)
            ref, tol = experts64(x, ids, w, g if gate else None, share if join else None)
            check_experts(torch_dev, got, ref, tol)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_experts_unbalanced(g9, torch_dev, dtype):
    """All tokens at one expert, none at the others; every place empty; an expert twice in a token's places."""
    r = np.random.default_rng(9)
    T, S, E, N, K = 150, 2, 12, 80, 300
    W, w = weights(r, torch_dev, g9, E, N, K)
    x = r.standard_normal((T, K)).astype(dtype)
    share = r.random((T, S)).astype(np.float32)
    for ids in (np.full((T, S), 7), np.full((T, S), -1), np.tile([[3, 3]], (T, 1)), np.tile([[11, 0]], (T, 1))):
        ids = ids.astype(np.int32)
        for join in (None, share):
            got = g9.moe_gemm(gpu(torch_dev, x), gpu(torch_dev, ids), W, weights=None if join is None else gpu(torch_dev, join))
            check_experts(torch_dev, got, *experts64(x, ids, w, None, join))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("T,S", [(1, 2), (8, 2), (20, 2), (60, 2), (100, 2)])
def test_experts_blocks_of_zeros_with_any_scale(g9, torch_dev, dtype, T, S):
    """Blocks and rows of zeros under any scale, NaN blocks beside them: few places without a plan, tiles of 16, 32 and 64 rows.
    X in steps of 2^-10: no sum of a row is rounded. Products of two such sums may be FP32 subnormals, of 2^-149 steps."""
    torch = torch_dev
    r = np.random.default_rng(T)
    E, K = 3, 640

    def experts():
        codes, scales = (np.stack(p) for p in zip(*(zero_block_rows(r, K) for _ in range(E))))
        return g9.mx4_load(gpu(torch, packed(codes)), gpu(torch, scales), K=K), values(codes, scales)

    (W, w), (G, g) = experts(), experts()
    nan = np.isnan(w).any((0, 2))           # the same rows of every expert
    ids = np.argsort(r.random((T, E)), 1)[:, :S].astype(np.int32)
    share = r.random((T, S)).astype(np.float32)
    x = (r.integers(-64, 65, (T, K)) / 1024).astype(dtype)
    for gate in (False, True):
        for join in (False, True):
            got = g9.moe_gemm(gpu(torch, x), gpu(torch, ids), W, gate=G if gate else None, weights=gpu(torch, share) if join else None)
            assert bool(got[..., gpu(torch, nan)].isnan().all())
            ref, tol = experts64(x, ids, w[:, ~nan], g[:, ~nan] if gate else None, share if join else None)
            check_experts(torch, got[..., gpu(torch, ~nan)], ref, tol + 2.0 ** -146)


@pytest.mark.parametrize("T", [3, 70])
def test_experts_ids_of_other_types(g9, torch_dev, T):
    """Ids of 64 bits, beyond 32 bits too, are no expert's unless they are 0..E-1; other integer types as they are."""
    torch = torch_dev
    r = np.random.default_rng(T)
    S, E, N, K = 6, 4, 40, 96
    W, w = weights(r, torch, g9, E, N, K)
    x = r.standard_normal((T, K)).astype(np.float32)
    ids = r.integers(0, E, (T, S))
    ids[:, 1], ids[:, 3] = 1 << 32, -(1 << 32) + 2
    ids[0, 0], ids[1, 2], ids[2, 5] = (1 << 31) + 1, np.iinfo(np.int64).min, np.iinfo(np.int64).max
    want = experts64(x, ids, w)
    assert (want[0][:, (1, 3)] == 0).all()
    check_experts(torch, g9.moe_gemm(gpu(torch, x), gpu(torch, ids), W), *want)
    check_experts(torch, torch.from_numpy(g9.moe_gemm(x, ids, W)), *want)
    small = r.integers(0, E, (T, S))
    for t in (torch.int64, torch.int16, torch.uint8):
        check_experts(torch, g9.moe_gemm(gpu(torch, x), gpu(torch, small).to(t), W), *experts64(x, small, w))


def test_experts_no_places(g9, torch_dev):
    """A token without places has nothing to join: its row of the result is zero."""
    torch = torch_dev
    W = g9.mx4_quantize(torch.ones((3, 40, 96), device="cuda"))
    ids, share = torch.empty((5, 0), dtype=torch.int32, device="cuda"), torch.empty((5, 0), device="cuda")
    for t in (torch.float16, torch.float32):
        x = torch.ones((5, 96), dtype=t, device="cuda")
        out = torch.full((7, 50), 3.0, dtype=t, device="cuda")
        assert g9.moe_gemm(x, ids, W, weights=share, C=out[1:6, 2:42]) is not None
        assert bool((out[1:6, 2:42] == 0).all())
        out[1:6, 2:42] = 3.0
        assert bool((out == 3.0).all())
        assert g9.moe_gemm(x, ids, W).shape == (5, 0, 40)
    assert (g9.moe_gemm(np.ones((5, 96), np.float32), np.empty((5, 0), np.int32), W, weights=np.empty((5, 0), np.float32)) == 0).all()
    L = g9._llm_library()
    C = torch.full((5, 40), 3.0, device="cuda")
    x = torch.ones((5, 96), device="cuda")
    call = lambda S, weights, C: L.gen9blas_moe_gemm(1, 5, S, None, x.data_ptr(), 96, 0, W._handle, None, weights, C, 40, 40)   # noqa: E731
    assert call(0, None, None) == 0 and call(0, None, C.data_ptr()) == 0 and call(0, x.data_ptr(), None) == -3
    torch.cuda.synchronize()
    assert bool((C == 3).all())
    assert call(0, x.data_ptr(), C.data_ptr()) == 0
    g9.flush()
    assert bool((C == 0).all())


def test_inputs_of_any_layout(g9, torch_dev):
    """Layouts that the C entry points do not take are copied: repeated and overlapping rows, permuted dimensions, NumPy's negative
    strides."""
    torch = torch_dev
    r = np.random.default_rng(6)
    E, S, N, K, T = 5, 3, 40, 96, 7
    W, _ = weights(r, torch, g9, E, N, K)
    ids = gpu(torch, np.argsort(r.random((T, E)), 1)[:, :S].astype(np.int32))
    share = gpu(torch, r.random((T, S)).astype(np.float32))
    for dtype in (torch.float16, torch.float32):
        x = gpu(torch, r.standard_normal((S, T, K))).to(dtype)
        flat = x.reshape(-1)
        for v in (x[0, :1].expand(T, K), flat.as_strided((T, K), (3, 1)), x.transpose(0, 1), x[:, :1].transpose(0, 1).expand(T, S, K),
                  x[0, :, None].expand(T, S, K), flat.as_strided((T, S, K), (K, 5, 1)), x[0].t().contiguous().t()):
            for kw in (dict(), dict(weights=share), dict(gate=W)):
                assert bool((g9.moe_gemm(v, ids, W, **kw) == g9.moe_gemm(v.contiguous(), ids, W, **kw)).all())
        logits = flat.as_strided((T, 8), (2, 1))
        for v in (logits, flat[:8].expand(T, 8)):
            got, want = g9.moe_route(v, 2), g9.moe_route(v.contiguous(), 2)
            assert bool((got[0] == want[0]).all()) and bool((got[1] == want[1]).all())
    x, l, b = (r.standard_normal(n).astype(np.float32) for n in ((T, K), (T, 8), 8))
    i, w = ids.cpu().numpy(), share.cpu().numpy()
    got = g9.moe_gemm(x[::-1, ::-1], i[::-1], W, weights=w[::-1, ::-1])
    assert np.array_equal(got, g9.moe_gemm(x[::-1, ::-1].copy(), i[::-1].copy(), W, weights=w[::-1, ::-1].copy()))
    got, want = g9.moe_route(l[:, ::-1], 2, bias=b[::-1]), g9.moe_route(l[:, ::-1].copy(), 2, bias=b[::-1].copy())
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_experts_of_many_places_and_columns(g9, torch_roomy):
    """2^18 places of 65536 columns: offsets past 32 bits, and more tiles of 16 columns than a launch takes (it has wider ones)."""
    torch = torch_roomy
    g = torch.Generator(device="cuda").manual_seed(1)
    T, E, N, K = 1 << 18, 2, 1 << 16, 32
    w = torch.randint(-2, 3, (E, N, K), generator=g, device="cuda").half()
    x = torch.randint(-2, 3, (T, K), generator=g, device="cuda").half()
    ids = torch.randint(0, E, (T, 1), generator=g, device="cuda", dtype=torch.int32)
    y = g9.moe_gemm(x, ids, g9.mx4_quantize(w))
    for e in range(E):
        for t in torch.nonzero(ids[:, 0] == e)[:, 0].split(4096):
            assert bool((y[t, 0] == x[t] @ w[e].t()).all())


@pytest.mark.parametrize("step", [256, 260, 262, 263])
def test_experts_rows_in_place(g9, torch_dev, step):
    """More than 40 places an expert, whole 128-k chunks of FP16: rows that the tile kernel copies to LDS from where they lie, at any
    multiple of four bytes, and those that go by way of the work space."""
    torch = torch_dev
    r = np.random.default_rng(step)
    T, S, E, N, K = 100, 2, 3, 300, 256
    W, w = weights(r, torch, g9, E, N, K)
    ids = np.argsort(r.random((T, E)), 1)[:, :S].astype(np.int32)
    flat = gpu(torch, r.standard_normal(T * (S + 1) * step + 8).astype(np.float16))
    for off in (0, 1, 2, 4, 6):
        for x in (flat.as_strided((T, K), (step, 1), off), flat.as_strided((T, 1, K), (step, step, 1), off).expand(T, S, K),
                  flat.as_strided((T, S, K), (S * step, step, 1), off), flat.as_strided((T, S, K), ((S + 1) * step, step, 1), off)):
            check_experts(torch, g9.moe_gemm(x, gpu(torch, ids), W), *experts64(x.cpu().numpy(), ids, w))


@pytest.mark.parametrize("T", [1, 5, 90])
def test_experts_strides(g9, torch_dev, T):
    """Rows of X and C with strides of tokens and places, at odd alignments; nothing written beside C; NaN in one token's row
    stays with it."""
    torch = torch_dev
    r = np.random.default_rng(T)
    S, E, N, K = 3, 6, 50, 140
    W, w = weights(r, torch, g9, E, N, K)
    ids = np.argsort(r.random((T, E)), 1)[:, :S].astype(np.int32)
    for dtype in (np.float16, np.float32):
        big = gpu(torch, r.standard_normal((T, S + 2, K + 5)).astype(dtype))
        x = big[:, 1:S + 1, 3:K + 3]
        out = torch.full((T, S + 1, N + 9), 5.0, dtype=big.dtype, device="cuda")
        g9.moe_gemm(x, gpu(torch, ids), W, C=out[:, :S, 1:N + 1])
        check_experts(torch, out[:, :S, 1:N + 1], *experts64(x.cpu().numpy(), ids, w))
        out[:, :S, 1:N + 1] = 5.0
        assert bool((out == 5.0).all())
        if T > 1:
            bad = x.clone()
            bad[0] = float("nan")
            got = g9.moe_gemm(bad, gpu(torch, ids), W)
            assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1:]).all())


def test_experts_layer(g9, torch_dev):
    """A whole layer as a program runs it, in no-wait mode: router, gated first products, joined second products; repeated
    calls give the same bits."""
    torch = torch_dev
    r = np.random.default_rng(1)
    E, S, D, F = 16, 4, 256, 320
    up, u = weights(r, torch, g9, E, F, D)
    gate, v = weights(r, torch, g9, E, F, D)
    down, d = weights(r, torch, g9, E, D, F)
    g9.set_nowait(True)
    try:
        for T in (1, 5, 64, 700):
            x = r.standard_normal((T, D)).astype(np.float16)
            logits = r.normal(0, 2, (T, E)).astype(np.float32)
            xd, ld = gpu(torch, x), gpu(torch, logits)
            runs = []
            for _ in range(3):
                ids, w = g9.moe_route(ld, S)
                h = g9.moe_gemm(xd, ids, up, gate=gate)
                runs.append((ids, w, h, g9.moe_gemm(h, ids, down, weights=w)))
            g9.flush()
            assert all(bool((a == b).all()) for a, b in zip(runs[0], runs[1])) and all(bool((a == b).all()) for a, b in zip(runs[0], runs[2]))
            ids, w, h, y = (t.cpu().numpy() for t in runs[0])
            check_experts(torch, runs[0][2], *experts64(x, ids, u, v))
            check_experts(torch, runs[0][3], *experts64(h, ids, d, None, w))
    finally:
        g9.set_nowait(False)


def test_refusals(g9, torch_dev):
    torch = torch_dev
    L = g9._llm_library()
    x = torch.zeros((4, 64), device="cuda")
    ids, w = torch.full((4, 2), 9, dtype=torch.int32, device="cuda"), torch.full((4, 2), 9.0, device="cuda")
    INVALID, UNSUPPORTED = -3, -2

    def route(type=1, T=4, E=64, logits=x.data_ptr(), ldl=64, bias=None, score=0, groups=1, top=1, k=2, ids=ids.data_ptr()):
        return L.gen9blas_moe_route(type, T, E, logits, ldl, bias, score, groups, top, k, 1, 1.0, ids, w.data_ptr())

    assert route(type=3) == UNSUPPORTED and route(score=2) == UNSUPPORTED
    for bad in (dict(E=0), dict(E=1025), dict(k=0), dict(k=65), dict(ldl=63), dict(groups=5), dict(groups=0), dict(groups=8, top=9), dict(top=0),
                dict(logits=None), dict(logits=np.zeros(256, np.float32).ctypes.data), dict(T=1 << 20), dict(ids=None)):
        assert route(**bad) == INVALID, bad
    assert route(T=0, logits=None) == 0
    torch.cuda.synchronize()
    assert bool((ids == 9).all()) and bool((w == 9).all())
    W = g9.mx4_quantize(torch.ones((3, 8, 64), device="cuda"))
    other = g9.mx4_quantize(torch.ones((3, 9, 64), device="cuda"))
    i = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    C = torch.full((4, 2, 8), 5.0, device="cuda")

    def gemm(type=1, T=4, S=2, i=i.data_ptr(), X=x.data_ptr(), ldt=64, lds=0, W=W._handle, gate=None, weights=None, C=C.data_ptr(), ldct=16, ldcs=8):
        return L.gen9blas_moe_gemm(type, T, S, i, X, ldt, lds, W, gate, weights, C, ldct, ldcs)

    assert gemm(type=2) == UNSUPPORTED
    for bad in (dict(W=None), dict(gate=other._handle), dict(ldt=63), dict(lds=63), dict(lds=64), dict(lds=-64), dict(ldct=15), dict(ldcs=7), dict(X=None),
                dict(i=None), dict(C=None), dict(T=1 << 20), dict(weights=np.ones(8, np.float32).ctypes.data)):
        assert gemm(**bad) == INVALID, bad
    assert gemm(T=0) == 0 and gemm(S=0) == 0
    torch.cuda.synchronize()
    assert bool((C == 5.0).all())
    with pytest.raises(ValueError):
        g9.moe_gemm(x, i[:3], W)
    with pytest.raises(ValueError):
        g9.moe_gemm(x, i, W, gate=other)
    with pytest.raises(ValueError):
        g9.moe_gemm(x, i, W, weights=torch.ones((4, 3), device="cuda"))
    with pytest.raises(KeyError):
        g9.moe_route(x, 2, score="relu")
    with pytest.raises(RuntimeError):
        g9.moe_route(x, 65)
