// Linear layers: Y = R + dropout(act(X·Wᵀ + b)) in one product (gen9blas_linear) and its gradients (gen9blas_linear_backward).
//
// The forward product runs on the library's own FP16 and FP32 kernels for direct global→LDS loads (hgemm_kernel.h,
// sgemm_kernel.h), a few rows on the ones that stream the weights (skinny_kernel.h) or share them (linear_rows_kernel.h: some dozens of
// rows, and 3 to 16 on large weights, takes_rows), with linear_epilogue.h in the place of alpha and beta: a product that is stored first, and read again for its bias, activation and residual, costs 2 passes more
// over M·N values. The gradients' two products are gen9blas_gemm's.
#include "llm.h"
#include "linear_epilogue.h"
#include "hgemm_kernel.h"
#include "hgemm_tiles.h"
#include "sgemm_kernel.h"
#include "sgemm_tiles.h"
#include "skinny_kernel.h"
#include "linear_rows_kernel.h"
#include "colsum.h"
#include <algorithm>

namespace g9llm {

struct HParams : g9::hg::Params { Epilogue<_Float16> epilogue; };
struct SParams : g9::sg::Params { Epilogue<float> epilogue; };
template <class T> struct FewParams : g9::sk::Params { Epilogue<T> epilogue; };

// Rows of K elements into rows of ldd, a multiple of 8 (zeros past K); a thread has eight of them.
template <class T>
__global__ void __launch_bounds__(256) pad_rows_kernel(const T *__restrict__ X, long long ldx, int K, T *__restrict__ D, int groups, long long total) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / groups;
        const int k = (int)(i % groups) * 8;
        float v[8];
        load_some<8>(X + r * ldx + k, K - k, v);
        store_some<8>(D + i * 8, 8, v);
    }
}
template <class T> static int pad_rows(const void *X, long long ldx, long long rows, int K, int ldd, int slot, const T **D) {
    void *d;
    const long long total = rows * (ldd / 8);
    G9_TRY(work_buffer("linear", slot, (size_t)total * 8 * sizeof(T), &d));
    hipLaunchKernelGGL((pad_rows_kernel<T>), dim3((unsigned)std::min(cdiv(total, 256), 32LL * num_cus)), dim3(256), 0, stream, (const T *)X, ldx, K, (T *)d, ldd / 8, total);
    G9_HIP(hipGetLastError());
    *D = (const T *)d;
    return 0;
}

static int check_grid(long long workgroups, int threads) {
    if (workgroups * threads > 0xffffffffLL) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "linear: more tiles than one launch can index");
    return 0;
}

// The partial sums of a split k, 64 MiB: what the FP16 and FP32 products of libgen9blas.so have.
constexpr size_t SPLIT_BYTES = 64u << 20;

template <g9::hgl::HgCfg G> static int launch_h(HParams p, int slices) {
    constexpr int KB = g9::hgl::KB;
    p.tiles_m = (int)cdiv(p.M, G.BM), p.tiles_n = (int)cdiv(p.N, G.BN);
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    const dim3 block(G.WM * G.WN * 64);
    G9_TRY(check_grid(tiles, (int)block.x));
    if (slices > 1) {
        p.kper = std::max((int)cdiv(cdiv(p.K, slices), KB) * KB, 2 * KB);
        const int ns = (int)cdiv(p.K, p.kper);
        constexpr int PER = G.BM * G.BN / 512;   // 512 elements a wave
        hipLaunchKernelGGL((g9::hg::hgemm_kernel<G.BM, G.BN, G.WM, G.WN, KB, G.NS, true, true, G.RA, true, true, g9::hg::Params>), dim3((unsigned)tiles, (unsigned)ns), block, 0, stream, p);
        G9_HIP(hipGetLastError());
        hipLaunchKernelGGL((g9::hg::split_sum<G.BM, G.BN, G.WM, G.WN, HParams>), dim3((unsigned)cdiv(tiles * PER, 4)), dim3(256), 0, stream, p, ns);
    } else {
        hipLaunchKernelGGL((g9::hg::hgemm_kernel<G.BM, G.BN, G.WM, G.WN, KB, G.NS, true, true, G.RA, true, false, HParams>), dim3((unsigned)tiles), block, 0, stream, p);
    }
    G9_HIP(hipGetLastError());
    return 0;
}
static int tiles_product(HParams &p) {
    using namespace g9::hgl;
    const Choice c = choose({p.M, p.N, p.K, 1, p.ldc, 0, 1}, SPLIT_BYTES, num_cus);
    if (c.slices > 1) G9_TRY(work_buffer("linear", SLOT_PART, SPLIT_BYTES, (void **)&p.P));
    switch (c.cfg) {
    case 0: return launch_h<CFG[0]>(p, c.slices);
    case 1: return launch_h<CFG[1]>(p, c.slices);
    case 3: return launch_h<CFG[3]>(p, c.slices);
    case 4: return launch_h<CFG[4]>(p, c.slices);
    case 5: return launch_h<CFG[5]>(p, c.slices);
    case 6: return launch_h<CFG[6]>(p, c.slices);
    }
    return launch_h<CFG[2]>(p, c.slices);
}

template <g9::sgl::SgCfg G> static int launch_s(SParams p, int slices) {
    p.tiles_m = (int)cdiv(p.M, G.BM), p.tiles_n = (int)cdiv(p.N, G.BN);
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    const dim3 block(G.WM * G.WN * 64);
    G9_TRY(check_grid(tiles, (int)block.x));
    if (slices > 1) {
        const int ns = g9::sgl::slices_of(p.K, slices, p.kper);
        constexpr int PER = G.BM * G.BN / 256;   // 256 elements a wave
        hipLaunchKernelGGL((g9::sg::sgemm_kernel<G.BM, G.BN, G.WM, G.WN, G.NS, true, true, G.BLK, 0, 0, false, true, true, g9::sg::Params>), dim3((unsigned)tiles, (unsigned)ns), block, 0, stream, p);
        G9_HIP(hipGetLastError());
        hipLaunchKernelGGL((g9::sg::split_sum<G.BM, G.BN, G.WM, G.WN, 0, SParams>), dim3((unsigned)cdiv(tiles * PER, 4)), dim3(256), 0, stream, p, ns, (int)tiles);
    } else {
        hipLaunchKernelGGL((g9::sg::sgemm_kernel<G.BM, G.BN, G.WM, G.WN, G.NS, true, true, G.BLK, 0, 0, false, true, false, SParams>), dim3((unsigned)tiles), block, 0, stream, p);
    }
    G9_HIP(hipGetLastError());
    return 0;
}
static int tiles_product(SParams &p) {
    using namespace g9::sgl;
    const Choice c = choose({p.M, p.N, p.K, 1}, SPLIT_BYTES, false, false, num_cus);
    if (c.slices > 1) G9_TRY(work_buffer("linear", SLOT_PART, SPLIT_BYTES, (void **)&p.P));
    switch (c.cfg) {
    case 1: return launch_s<CFG[1]>(p, c.slices);
    case 3: return launch_s<CFG[3]>(p, c.slices);
    case 4: return launch_s<CFG[4]>(p, c.slices);
    }
    return launch_s<CFG[2]>(p, c.slices);
}

// Up to 16 rows: the weights streamed once, as gen9blas_gemm's few rows are (skinny.hip has what chose the shapes).
template <class T> static int few_rows(const FewParams<T> &p, bool vec) {
    auto run = [&](auto kernel, auto vkernel, int rows, int waves) -> int {
        const long long wgs = cdiv(p.N, rows);
        G9_TRY(check_grid(wgs, waves * 64));
        hipLaunchKernelGGL(vec ? vkernel : kernel, dim3((unsigned)wgs), dim3(waves * 64), 0, stream, p);
        G9_HIP(hipGetLastError());
        return 0;
    };
#define G9_FEW(MT, RW, KS, NC) run(g9::sk::skinny_kernel<T, MT, RW, KS, NC, false, FewParams<T>>, g9::sk::skinny_kernel<T, MT, RW, KS, NC, true, FewParams<T>>, RW, KS)
    if constexpr (sizeof(T) == 2) {
        if (p.M > 2 && vec && p.K % 256 == 0 && (p.swn + p.sam) * 32 < (1LL << 32)) {
            auto mfma = [&](auto kernel) { return run(kernel, kernel, 16, 2); };
            if (p.M <= 4) return mfma(g9::sk::skinny_mfma_kernel<4, 2, 4, FewParams<T>>);
            if (p.M <= 8) return mfma(g9::sk::skinny_mfma_kernel<8, 2, 4, FewParams<T>>);
            return mfma(g9::sk::skinny_mfma_kernel<16, 2, 3, FewParams<T>>);
        }
    }
    if (p.M <= 1) return G9_FEW(1, 1, 4, 2);
    if (p.M <= 2) return G9_FEW(2, 2, 4, 1);
    if (p.M <= 4) return G9_FEW(4, 4, 8, 1);
    if (p.M <= 8) return G9_FEW(8, 4, 4, 1);
    return G9_FEW(16, 8, 4, 1);
#undef G9_FEW
}

template <class T, int MT, int NS> static int some_rows(RowsArgs<T> a) {
    const long long tiles = cdiv(a.N, 64);
    const int pieces = (int)cdiv(a.K, 512 / sizeof(T));
    a.per = (int)cdiv(pieces, std::max(1LL, std::min<long long>(pieces, num_cus / tiles)));
    a.slices = (int)cdiv(pieces, a.per);
    if (a.slices > 1) G9_TRY(work_buffer("linear", SLOT_PART, (size_t)a.slices * tiles * 4 * MT * 1024, (void **)&a.parts));
    G9_TRY(check_grid(tiles * a.slices, 512));
    hipLaunchKernelGGL((linear_rows_kernel<T, MT, NS>), dim3((unsigned)(tiles * a.slices)), dim3(512), 0, stream, a);
    G9_HIP(hipGetLastError());
    if (a.slices > 1) hipLaunchKernelGGL((linear_rows_sum_kernel<T, MT>), dim3((unsigned)(tiles * MT)), dim3(256), 0, stream, a, (int)tiles);
    G9_HIP(hipGetLastError());
    return 0;
}

// Whether linear_rows_kernel takes M rows, by what it and the others measure (µs, it / others).
// - FP32 up to 64 rows, of 8 M weights: 32 × 4096 × 2048 (at 4 M alike) and 16 × 8192 × 1024 13 / 19, 32 × 4096 × 11008 45 / 65, 64 of them
//   60 / 67, 5 to 8 rows from 32 M on, 8 × 11008 × 4096 33 / 41. Not 4 × 4096 × 11008 41 / 34, nor more than 48 rows where the columns
//   alone make as many workgroups as there can be, and leave CUs without one: 64 × 11008 × 4096 78 / 67.
// - FP16 up to 32 rows, of 32 M weights: 32 × 4096 × 11008 23 / 25, 32 × 11008 × 4096 20.6 / 24.1 (32 × 4096 × 4096 13 / 13); up to 16, which
//   the streaming kernel takes without a second one, only where no slices of k are needed: 16 × 11008 × 4096 18.5 / 22.7, but 16 × 4096 ×
//   11008 21.7 / 19.2.
template <class T> static bool takes_rows(int M, int N, int K) {
    const long long weights = (long long)N * K;
    const bool alone = cdiv(N, 64) * 2 > num_cus;   // one slice of k
    if (sizeof(T) == 4) return weights >= (M > 8 ? 8 << 20 : 32 << 20) && M > 4 && M <= (alone ? 48 : 64);
    return weights >= 32 << 20 && M <= 32 && (M > 16 || (alone && M > 2));
}

template <class T>
static int linear(int M, int N, int K, const T *X, long long ldx, const T *W, long long ldw, const Epilogue<T> &e, T *Y, long long ldy) {
    constexpr int KB = sizeof(T) == 2 ? g9::hgl::KB : g9::sgl::KB;
    // The kernels on direct copies take one k-step of k or more, FP16 operands at 4-byte alignment with even row strides, and rows
    // of a tile within 4 GiB; for these, others are copied first, and a short k is filled up with zeros.
    auto copied = [&](const T *p, long long ld) { return K < KB || ld * 256 * (long long)sizeof(T) >= 1LL << 32 || (sizeof(T) == 2 && ((uintptr_t)p % 4 || ld % 2)); };
    const bool cx = copied(X, ldx), cw = copied(W, ldw), some = M <= 64 && takes_rows<T>(M, N, K);
    if (M <= 16 && (!some || cx || cw)) {
        FewParams<T> p{};
        p.a = X, p.w = W, p.C = Y, p.sam = ldx, p.swn = ldw, p.scm = ldy, p.scn = 1, p.M = M, p.N = N, p.K = K, p.epilogue = e;
        constexpr int V = 16 / sizeof(T);
        return few_rows<T>(p, (uintptr_t)X % 16 == 0 && (uintptr_t)W % 16 == 0 && ldx % V == 0 && ldw % V == 0);
    }
    const int Kp = K < KB ? KB : K, ldp = (int)cdiv(Kp, 8) * 8;
    if (cx) {
        G9_TRY(pad_rows(X, ldx, M, K, ldp, SLOT_X, &X));
        ldx = ldp;
    }
    if (cw) {
        G9_TRY(pad_rows(W, ldw, N, K, ldp, SLOT_W, &W));
        ldw = ldp;
    }
    if (some) {
        const RowsArgs<T> a = {X, W, Y, ldx, ldw, ldy, M, N, Kp, 1, 0, nullptr, e};
        if (M <= 16) return some_rows<T, 1, 3>(a);
        if (M <= 32) return some_rows<T, 2, 3>(a);
        if constexpr (sizeof(T) == 4) return M <= 48 ? some_rows<T, 3, 2>(a) : some_rows<T, 4, 2>(a);
    }
    std::conditional_t<sizeof(T) == 2, HParams, SParams> p{};
    p.A = X, p.B = W, p.C = Y, p.lda = ldx, p.ldb = ldw, p.ldc = ldy, p.M = M, p.N = N, p.K = Kp, p.alpha = 1.f, p.epilogue = e;
    // FP16 rows of whole 128-byte lines go out past the caches, where nothing reads them soon; parts of lines would take longer so (4096 ×
    // 11008 × 1024 97 µs, through the caches 113; 4096 × 11001 × 1024 149 and 132)
    auto lines = [](const T *q, long long ld) { return (uintptr_t)q % 128 == 0 && ld % 64 == 0; };
    p.epilogue.past = sizeof(T) == 2 && lines(Y, ldy) && (!e.Z || lines(e.Z, e.ldz));
    return tiles_product(p);
}

// dZ = dropout(act'(Z) · dY) and, for each block of `rows` rows, the sums of its columns (before they are rounded). A workgroup
// has 2^cols threads side by side, eight columns each, and the others below them, each with every (256 >> cols)th row of the
// block, four of them on their way at once. dZ and Z may be null (no activation: dZ = dropout(dY)).
template <class T, int KIND>
__global__ void __launch_bounds__(256) linear_back_kernel(const T *__restrict__ dY, long long lddy, const T *__restrict__ Z, long long ldz, Activation act, Dropout d,
                                                          int M, int N, int rows, int cols, T *__restrict__ dZ, long long lddz, float *__restrict__ sums) {
    constexpr int V = 8, U = 4;
    __shared__ float part[256][V + 1];
    const int ct = 1 << cols, c = threadIdx.x & (ct - 1), r = threadIdx.x >> cols, step = 256 >> cols, n = ((blockIdx.x << cols) + c) * V, valid = N - n;
    const long long block = blockIdx.y, m0 = block * rows, m1 = min(m0 + rows, (long long)M);
    float sum[V] = {};
    auto row = [&](long long m, float *v, const float *z) {
        if (Z)
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = gradient<T, KIND>(act, v[e], z[e]);
        if (d.limit) drop<V>(d, (unsigned)m, n, v);   // last: what is dropped is zero, whatever Z is there
        if (dZ) store_some<V>(dZ + m * lddz + n, valid, v);
#pragma unroll
        for (int e = 0; e < V; e++) sum[e] += v[e];
    };
    long long m = m0 + r;
    if (valid >= V) {
        for (; m + (U - 1) * step < m1; m += U * step) {
            float v[U][V], z[U][V];
#pragma unroll
            for (int u = 0; u < U; u++) {
                load_some<V>(dY + (m + u * step) * lddy + n, V, v[u]);
                if (Z) load_some<V>(Z + (m + u * step) * ldz + n, V, z[u]);
            }
#pragma unroll
            for (int u = 0; u < U; u++) row(m + u * step, v[u], z[u]);
        }
    }
    if (valid > 0)
        for (; m < m1; m += step) {
            float v[V], z[V];
            load_some<V>(dY + m * lddy + n, valid, v);
            if (Z) load_some<V>(Z + m * ldz + n, valid, z);
            row(m, v, z);
        }
    if (!sums) return;
#pragma unroll
    for (int e = 0; e < V; e++) part[threadIdx.x][e] = sum[e];
    __syncthreads();
    if (r || valid <= 0) return;
    for (int i = 1; i < step; i++)
#pragma unroll
        for (int e = 0; e < V; e++) sum[e] += part[(i << cols) + c][e];
    store_some<V>(sums + block * N + n, valid, sum);
}

template <class T>
static int backward(int type, int M, int N, int K, const T *dY, int lddy, const T *Z, int ldz, int act, const Dropout &d, const T *X, int ldx, const T *W, int ldw,
                    T *dX, int lddx, T *dW, int lddw, float *db, int accumulate) {
    // gen9blas_gemm has its slower kernel for FP16 operands with odd row strides or addresses: where the product is long enough
    // to pay for it, they are copied (gradients of 2685 × 4952 × 1081 132 µs, as they lie 230; 128 × 4096 × 4097 68 and 80, 64 rows 75
    // and 72)
    constexpr int LONG = 128;
    auto odd = [&](const T *p, int ld) { return sizeof(T) == 2 && (ld % 2 || (uintptr_t)p % 4); };
    // without an activation or dropout dZ is dY itself. Otherwise it is rounded to the type, once, for the two products (db adds it up
    // before): FP16 2^-11 of a value, so that dX and dW are off by 2.9e-4 of their size instead of 2.1e-4, their own rounding's (2048 × 11008 ×
    // 4096, GELU). Products of FP32 dZ run on the FP32 matrix cores, at a ninth of the rate; dZ as the sum of two FP16 numbers takes
    // twice the products.
    const bool own = act || d.limit || (odd(dY, lddy) && M >= LONG && K >= LONG && (dX || dW));
    const int lddz = own ? (int)cdiv(N, 8) * 8 : lddy;
    T *dZ = nullptr;
    void *p;
    if (own && (dX || dW)) {
        G9_TRY(work_buffer("linear_backward", SLOT_DZ, (size_t)M * lddz * sizeof(T), &p));
        dZ = (T *)p;
    }
    float *sums = nullptr;
    const int rows = (int)std::max(64LL, cdiv(M, 512));
    const long long blocks = cdiv(M, rows);
    if (db) {
        G9_TRY(work_buffer("linear_backward", SLOT_SUMS, (size_t)blocks * N * 4, &p));
        sums = (float *)p;
    }
    // copies and their buffers come before a result is written: a call that lacks the memory leaves a db that it would be added to
    if (dX && odd(W, ldw) && M >= LONG) {
        const int ldp = (int)cdiv(K, 8) * 8;
        G9_TRY(pad_rows(W, ldw, N, K, ldp, SLOT_W, &W));
        ldw = ldp;
    }
    if (dW && odd(X, ldx) && N >= LONG) {
        const int ldp = (int)cdiv(K, 8) * 8;
        G9_TRY(pad_rows(X, ldx, M, K, ldp, SLOT_X, &X));
        ldx = ldp;
    }
    if (dZ || db) {
        const Activation a = make_act(act);
        int cols = 0;
        while (cols < 5 && (8 << cols) < N) cols++;
        const dim3 grid((unsigned)cdiv(N, 8 << cols), (unsigned)blocks);
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, dY, lddy, act ? Z : nullptr, ldz, a, d, M, N, rows, cols, dZ, lddz, sums);
        };
        if (a.kind == KIND_CLIP) run(linear_back_kernel<T, KIND_CLIP>);
        else if (a.kind == KIND_SIGMOID) run(linear_back_kernel<T, KIND_SIGMOID>);
        else run(linear_back_kernel<T, KIND_ERF>);
        G9_HIP(hipGetLastError());
        if (db) G9_TRY(column_sums(sums, blocks, N, N, db, nullptr, accumulate));
    }
    const T *g = own ? dZ : dY;
    auto product = [&](int tA, int m, int n, int k, const void *A, int lda, const void *B, int ldb, double beta, void *C, int ldc) -> int {
        if (int r = gen9blas_gemm(type, tA, 0, m, n, k, 1.0, A, lda, B, ldb, beta, C, ldc)) return fail(r, "%s", gen9blas_error());
        return 0;
    };
    if (dX) G9_TRY(product(0, M, K, N, g, lddz, W, ldw, 0.0, dX, lddx));
    if (dW) G9_TRY(product(1, N, K, M, g, lddz, X, ldx, accumulate ? 1.0 : 0.0, dW, lddw));
    return 0;
}

}  // namespace g9llm

using namespace g9llm;

static bool known(int type) { return type == GEN9BLAS_H || type == GEN9BLAS_S; }
constexpr int LONGEST_K = 1 << 22;   // 256 rows of FP16 or FP32 within 4 GiB
// Kernels count rows and columns in an int, up to the end of the last tile.
static int countable(int M, int N, const char *who) {
    if (M > 0x7ffff000 || N > 0x7ffff000) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "%s: more rows or columns than kernels count (M %d, N %d)", who, M, N);
    return 0;
}

extern "C" {

int gen9blas_linear(int type, int M, int N, int K, const void *X, int ldx, const void *W, int ldw, const float *bias, int act, void *Z, int ldz, double p,
                    uint64_t seed, uint64_t offset, const void *R, int ldr, void *Y, int ldy) {
    G9_TRY(begin());
    if (!known(type)) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "linear: type %d unavailable", type);
    if (act < GEN9BLAS_ACT_NONE || act > GEN9BLAS_ACT_SILU) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "linear: activation %d unavailable", act);
    if (!(p >= 0 && p <= 1)) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "linear: dropout %g is not in [0, 1]", p);
    if (M <= 0 || N <= 0) return 0;
    if (K < 1 || ldx < K || ldw < K || ldy < N || (Z && ldz < N) || (R && ldr < N))
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "linear: M %d, N %d, K %d, ldx %d, ldw %d, ldz %d, ldr %d, ldy %d", M, N, K, ldx, ldw, ldz, ldr, ldy);
    G9_TRY(countable(M, N, "linear"));
    if (K >= LONGEST_K) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "linear: rows of %d values; the longest have %d", K, LONGEST_K - 1);
    const size_t es = elem_size(type);
    G9_TRY(need_device(X, ((size_t)(M - 1) * ldx + K) * es, "linear: X"));
    G9_TRY(need_device(W, ((size_t)(N - 1) * ldw + K) * es, "linear: W"));
    if (bias) G9_TRY(need_device(bias, (size_t)N * 4, "linear: bias"));
    if (Z) G9_TRY(need_device(Z, ((size_t)(M - 1) * ldz + N) * es, "linear: Z"));
    if (R) G9_TRY(need_device(R, ((size_t)(M - 1) * ldr + N) * es, "linear: R"));
    G9_TRY(need_device(Y, ((size_t)(M - 1) * ldy + N) * es, "linear: Y"));
    const Activation a = make_act(act);
    const Dropout d = make_dropout(p, seed, offset);
    typedef _Float16 H;
    if (type == GEN9BLAS_H) return linear<H>(M, N, K, (const H *)X, ldx, (const H *)W, ldw, {bias, (H *)Z, (const H *)R, ldz, ldr, a, d}, (H *)Y, ldy);
    return linear<float>(M, N, K, (const float *)X, ldx, (const float *)W, ldw, {bias, (float *)Z, (const float *)R, ldz, ldr, a, d}, (float *)Y, ldy);
}

int gen9blas_linear_backward(int type, int M, int N, int K, const void *dY, int lddy, const void *Z, int ldz, int act, double p, uint64_t seed, uint64_t offset,
                             const void *X, int ldx, const void *W, int ldw, void *dX, int lddx, void *dW, int lddw, float *db, int accumulate) {
    G9_TRY(begin());
    if (!known(type)) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "linear_backward: type %d unavailable", type);
    if (act < GEN9BLAS_ACT_NONE || act > GEN9BLAS_ACT_SILU) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "linear_backward: activation %d unavailable", act);
    if (!(p >= 0 && p <= 1)) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "linear_backward: dropout %g is not in [0, 1]", p);
    if (N <= 0 || (!dX && !dW && !db)) return 0;
    M = std::max(M, 0);
    if (K < 1 || lddy < N || (act && ldz < N) || (dW && (ldx < K || lddw < K)) || (dX && (ldw < K || lddx < K)))
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "linear_backward: M %d, N %d, K %d, lddy %d, ldz %d, ldx %d, ldw %d, lddx %d, lddw %d", M, N, K, lddy, ldz, ldx, ldw, lddx, lddw);
    G9_TRY(countable(M, N, "linear_backward"));
    const size_t es = elem_size(type);
    if (M) {
        G9_TRY(need_device(dY, ((size_t)(M - 1) * lddy + N) * es, "linear_backward: dY"));
        if (act) G9_TRY(need_device(Z, ((size_t)(M - 1) * ldz + N) * es, "linear_backward: Z"));
        if (dW) G9_TRY(need_device(X, ((size_t)(M - 1) * ldx + K) * es, "linear_backward: X"));
        if (dX) G9_TRY(need_device(W, ((size_t)(N - 1) * ldw + K) * es, "linear_backward: W"));
        if (dX) G9_TRY(need_device(dX, ((size_t)(M - 1) * lddx + K) * es, "linear_backward: dX"));
    }
    if (dW) G9_TRY(need_device(dW, ((size_t)(N - 1) * lddw + K) * es, "linear_backward: dW"));
    if (db) G9_TRY(need_device(db, (size_t)N * 4, "linear_backward: db"));
    if (!M) {   // sums over no rows
        if (accumulate) return 0;
        if (dW) G9_TRY(zero_rows(dW, (long long)lddw * es, N, (long long)K * es));
        return db ? zero_rows(db, 4LL * N, 1, 4LL * N) : 0;
    }
    G9_TRY(not_captured("linear_backward"));   // the products' library has buffers of its own
    const Dropout d = make_dropout(p, seed, offset);
    typedef _Float16 H;
    if (type == GEN9BLAS_H)
        return backward<H>(type, M, N, K, (const H *)dY, lddy, (const H *)Z, ldz, act, d, (const H *)X, ldx, (const H *)W, ldw, (H *)dX, lddx, (H *)dW, lddw, db, accumulate);
    return backward<float>(type, M, N, K, (const float *)dY, lddy, (const float *)Z, ldz, act, d, (const float *)X, ldx, (const float *)W, ldw, (float *)dX, lddx, (float *)dW, lddw, db, accumulate);
}

}  // extern "C"
