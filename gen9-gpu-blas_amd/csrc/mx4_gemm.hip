// gen9blas_mx4_gemm and gen9blas_mx4_gemm_q: products of FP16, FP32 or MX4 rows with MX4 weights.
#include "mx4_tile_kernel.h"
#include "mx4_q_kernel.h"
#include "mx4_rows_kernel.h"

namespace g9llm {

// Both operands MX4, few rows: a workgroup makes a tile of 16 rows × 16 columns, its 4 waves every fourth group of 512 k.
// The operands go to the matrix cores as they lie, both read by every tile (W once from memory, then from L2): few rows leave the time to
// latency, and the many small workgroups hide it.
template <class O>
__global__ void __launch_bounds__(256) mx4_gemm_q_few_kernel(Mx4View A, Mx4View W, O *__restrict__ C, long long ldc, int mtiles, int) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    if ((int)blockIdx.x >= mtiles * W.rt) return;
    const int nt = blockIdx.x % W.rt, mt = blockIdx.x / W.rt;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const u32x4 *ac = reinterpret_cast<const u32x4 *>(A.codes) + (long long)mt * A.kc * 64 + lane;
    const u32x4 *wc = reinterpret_cast<const u32x4 *>(W.codes) + (long long)nt * W.kc * 64 + lane;
    const int *as = reinterpret_cast<const int *>(A.scales) + (long long)mt * A.kg * 64 + lane;
    const int *ws = reinterpret_cast<const int *>(W.scales) + (long long)nt * W.kg * 64 + lane;
    for (int grp = wv; grp < W.kg; grp += 4) {
        const int sa = as[grp * 64], sw = ws[grp * 64];
        auto step = [&](auto J) {
            constexpr int j = decltype(J)::value;
            const int c = grp * 4 + j;
            if (c >= W.kc) return;
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(wc[(long long)c * 64]), fp4_operand(ac[(long long)c * 64]), acc, 4, 4, j, sw, j, sa);
        };
        step(std::integral_constant<int, 0>());
        step(std::integral_constant<int, 1>());
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    }
    __shared__ f32x4 part[3][64];
    if (wv) part[wv - 1][lane] = acc;
    __syncthreads();
    if (wv) return;
#pragma unroll
    for (int w = 0; w < 3; w++) acc += part[w][lane];
    const int row = mt * 16 + r, n = nt * 16 + 4 * g;
    if (row >= A.rows) return;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (n + j < W.rows) C[row * ldc + n + j] = (O)acc[j];
}

template <class O> static int launch_q(const Mx4View &A, const Mx4View &W, O *C, long long ldc) {
    auto run = [&](auto kernel, int rows, int cols) -> int {   // of row tiles
        const long long mtiles = cdiv(A.rt, rows), ntiles = cdiv(W.rt, cols), wgs = cdiv(mtiles * ntiles, 8) * 8;
        if (wgs > 0xffffff) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm_q: more tiles than one launch can index");
        hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(256), 0, stream, A, W, C, ldc, (int)mtiles, (int)ntiles);
        G9_HIP(hipGetLastError());
        return 0;
    };
    // µs with the quantisation of A's rows: few kernel 100 × 4096 × 4096 11.3 and 100 × 4096 × 11008 17.5, ring kernel 12.8 and 21.8;
    // 64 × 11008 × 4096 and 200 × 4096 × 4096 15.1 and 15.8, ring kernel 13.0 and 13.2
    if ((long long)A.rt * W.rt <= 8 * num_cus) return run(mx4_gemm_q_few_kernel<O>, 1, 1);
    // ring kernel 2000 × 6000 × 4096 (192 tiles of 256 × 256) 38.5, tile kernel 39.3; 2300 × 6100 × 4096 (216) 45.7 and 42.8,
    // 3000 × 5000 × 4096 (240) 50.3 and 42.6
    if (cdiv(A.rt, 16) * cdiv(W.rt, 16) * 5 < 4 * num_cus) return run(mx4_gemm_q_ring_kernel<O>, 8, 8);
    return run(mx4_gemm_q_tile_kernel<O>, 16, 16);
}

static int split_space(const Rows &R, const Mx4View &W, Split *s) {
    s->rows = R.M, s->ld = (long long)W.rt * 16;
    return scratch(SLOT_PART, (size_t)s->parts * s->rows * s->ld * 4, (void **)&s->sums);
}
template <class O> static int sum_parts(const Rows &R, const Mx4View &W, const Split &split) {
    if (split.parts > 1)
        hipLaunchKernelGGL((mx4_sum_parts_kernel<O>), dim3((unsigned)cdiv(split.rows * split.ld, 256)), dim3(256), 0, stream, R, split, W.rows);
    G9_HIP(hipGetLastError());
    return 0;
}

// Up to 16 rows in tiles of 16 columns; k is split until there is about a workgroup a CU.
template <class T> static int launch_rows(const Rows &R, const Mx4View &W) {
    Split split = {1, nullptr, 0, 0};
    const int ways = num_cus / W.rt, most = W.kc / 8;
    if (ways > 1 && most > 1) {
        split.parts = ways < most ? ways : most;
        G9_TRY(split_space(R, W, &split));
    }
    if ((long long)W.rt * split.parts > 0xffffff) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm: more tiles than one launch can index");
    hipLaunchKernelGGL((mx4_gemm_rows_kernel<T, T, 4, false, false>), dim3((unsigned)(W.rt * split.parts)), dim3(256), 0, stream, R, W, W, 1, split);
    G9_HIP(hipGetLastError());
    return sum_parts<T>(R, W, split);
}

// Tiles of MT·16 rows × 128·NT columns; k is split until there is about a workgroup a CU.
template <class T, int MT, int NT, int D> static int launch_few(const Rows &R, const Mx4View &W) {
    const int ntiles = (int)cdiv(W.rt, NT * 8), mtiles = (int)cdiv(R.M, MT * 16);
    const long long tiles = (long long)mtiles * ntiles;
    Split split = {1, nullptr, 0, 0};
    const int ways = (int)(num_cus / tiles), most = W.kc / 4;
    if (ways > 1 && most > 1) {
        split.parts = ways < most ? ways : most;
        G9_TRY(split_space(R, W, &split));
    }
    if (tiles * split.parts > 0x7fffff) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm: more tiles than one launch can index");
    hipLaunchKernelGGL((mx4_gemm_few_kernel<T, T, MT, NT, D, false, false>), dim3((unsigned)(cdiv(tiles * split.parts, 8) * 8)), dim3(512), 0, stream, R, W, W, 1, mtiles, ntiles, split);
    G9_HIP(hipGetLastError());
    return sum_parts<T>(R, W, split);
}

// Tiles of 64 rows × 256 columns.
template <class T> static int launch_tiles(const Rows &R, const Mx4View &W) {
    Planes A;
    G9_TRY(stage_planes<T>(R, R.M, W.K, W.kc, &A));
    const long long mtiles = cdiv(R.M, 64), ntiles = cdiv(W.rt, 16);
    if (mtiles * ntiles > 0xfffff0) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm: more tiles than one launch can index");
    hipLaunchKernelGGL((mx4_gemm_tile_kernel<T, T, false, false>), dim3((unsigned)(cdiv(mtiles * ntiles, 8) * 8)), dim3(256), 0, stream, A, R, W, W, 1, (int)mtiles,
                       (int)ntiles);
    G9_HIP(hipGetLastError());
    return 0;
}

template <class T> static int launch_dense(const Rows &R, const Mx4View &W) {
    constexpr bool F = sizeof(T) == 4;
    if (R.M <= 16) {
        // FP32 rows are taken apart once a workgroup in the few kernel, once a wave in the rows kernel: 8 × 4096 × 11008 10.7 µs and 13.2
        if constexpr (F) return launch_few<T, 1, 2, 4>(R, W);
        // FP16: each 16 columns of the rows kernel read all rows again, from L2; the few kernel, eight times as wide, splits k where it has
        // fewer workgroups than CUs, and a second launch adds the parts. µs a call, rows kernel and few kernel: 1 × 11008 × 4096
        // 9.2 and 10.7, 8 × 11008 × 4096 (`again`, the elements read, 23 M) 11.1 and 11.1, 16 × 4096 × 8192 (34 M) 11.0 and 10.4,
        // 16 × 11008 × 4096 (45 M) 15.2 and 11.6. Where the rows kernel splits k too: 4 × 2048 × 8192 (4 M) 7.9 and 8.3, 8 × 2048 × 8192
        // (8 M) 8.5 and 8.3, 16 × 2048 × 8192 (17 M) 10.2 and 8.6. Where the few kernel need not: 1 × 16384 × 4096 (split) 11.5 and 11.9,
        // 1 × 17000 × 4096 (whole) 13.0 and 12.0, 16 × 22016 × 4096 27.0 and 12.6.
        const long long again = (long long)W.rt * W.K * R.M;
        const bool few_whole = cdiv(W.rt, 8) * 2 > num_cus, rows_whole = W.rt * 2 > num_cus;
        if (!few_whole && again <= (rows_whole ? 26000000 : 8000000)) return launch_rows<T>(R, W);
        return launch_few<T, 1, 1, 4>(R, W);
    }
    // 128 columns a workgroup; with 256, which reads the rows from LDS half as often but leaves twice the parts to be summed or half
    // the workgroups, µs a call: FP32 24 × 4096 × 11008 17.8 and 19.0, 24 × 11008 × 4096 20.2 and 19.1, 28 × 2048 × 2048 9.5 and 11.8; FP16
    // 24 × 4096 × 11008 13.0 and 15.1, 24 × 11008 × 4096 12.5 and 14.2
    if (R.M <= 32) return launch_few<T, 2, 1, 4>(R, W);
    // 64 rows: 128 columns, 256 columns, or the tile kernel, which has 64 × 256 too but fills the GPU with 768 workgroups, not 256.
    // FP16 512 × 4096 × 4096 (256 workgroups of 128 columns) 24.8, 29.1 and 33.1 µs, 1000 × 4096 × 4096 (512) 42.7, 37.1 and 40.5,
    // 400 × 11008 × 4096 (301 of 256 columns) 55.2, 65.0 and 54.8. FP32, where LDS gives three pieces of the rows: 100 × 4096 × 4096 (64 of 128
    // columns) 23.6, 25.6 and 26.6, 192 × 4096 × 4096 (96) 36.3, 30.8 and 36.0, 1000 × 4096 × 4096 (256 of 256 columns) 121, 87 and 98,
    // 400 × 11008 × 4096 156, 148 and 124.
    const long long mtiles = cdiv(R.M, 64);
    if (mtiles * cdiv(W.rt, 8) <= num_cus / (F ? 3 : 1)) return launch_few<T, 4, 1, 2>(R, W);
    if (mtiles * cdiv(W.rt, 16) <= num_cus) return launch_few<T, 4, 2, 2>(R, W);
    return launch_tiles<T>(R, W);
}

}  // namespace g9llm

using namespace g9llm;

extern "C" {

int gen9blas_mx4_gemm(int type, int M, const void *A, int lda, const gen9blas_mx4 *W, void *C, int ldc) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm: type %d unavailable", type);
    if (!W || W->count != 1) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_gemm: %s", W ? "W holds several matrices" : "no W");
    if (M <= 0) return 0;
    if (lda < W->K || ldc < W->rows) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_gemm: lda %d < K %d or ldc %d < N %d", lda, W->K, ldc, W->rows);
    const int es = elem_size(type);
    G9_TRY(need_device(A, ((size_t)(M - 1) * lda + W->K) * es, "mx4_gemm: A"));
    G9_TRY(need_device(C, ((size_t)(M - 1) * ldc + W->rows) * es, "mx4_gemm: C"));
    const Rows R = {A, C, lda, 0, ldc, 0, M, 1, nullptr, nullptr, nullptr, nullptr};
    return type == GEN9BLAS_H ? launch_dense<_Float16>(R, view(W)) : launch_dense<float>(R, view(W));
}

int gen9blas_mx4_gemm_q(int type, const gen9blas_mx4 *A, const gen9blas_mx4 *W, void *C, int ldc) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm_q: type %d unavailable", type);
    if (!A || !W || A->count != 1 || W->count != 1) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_gemm_q: %s", A && W ? "an operand holds several matrices" : "no A or no W");
    if (A->K != W->K || ldc < W->rows) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_gemm_q: K %d and %d, ldc %d, N %d", A->K, W->K, ldc, W->rows);
    G9_TRY(need_device(C, ((size_t)(A->rows - 1) * ldc + W->rows) * elem_size(type), "mx4_gemm_q: C"));
    return type == GEN9BLAS_H ? launch_q<_Float16>(view(A), view(W), (_Float16 *)C, ldc) : launch_q<float>(view(A), view(W), (float *)C, ldc);
}

}  // extern "C"
