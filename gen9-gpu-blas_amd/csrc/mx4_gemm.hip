// gen9blas_mx4_gemm and gen9blas_mx4_gemm_q: products of FP16, FP32 or MX4 rows with MX4 weights.
#include "mx4_tile_kernel.h"
#include "mx4_q_kernel.h"
#include "mx4_rows_kernel.h"

namespace g9llm {

// Both operands MX4, any shape: a workgroup makes 64 rows × 16 columns, its 4 waves every fourth group of 512 k.
template <class O>
__global__ void __launch_bounds__(256) mx4_gemm_q_any_kernel(Mx4View A, Mx4View W, O *__restrict__ C, long long ldc, int mtiles, int) {
    constexpr int MT = 4;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    if ((int)blockIdx.x >= mtiles * W.rt) return;
    const int nt = blockIdx.x % W.rt, mt = blockIdx.x / W.rt * MT;
    f32x4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32x4 *wc = reinterpret_cast<const u32x4 *>(W.codes) + (long long)nt * W.kc * 64 + lane;
    const int *ws = reinterpret_cast<const int *>(W.scales) + (long long)nt * W.kg * 64 + lane;
    for (int grp = wv; grp < W.kg; grp += 4) {
        const int sw = ws[grp * 64];
        int sa[MT];
#pragma unroll
        for (int m = 0; m < MT; m++)
            sa[m] = reinterpret_cast<const int *>(A.scales)[((long long)min(mt + m, A.rt - 1) * A.kg + grp) * 64 + lane];
        auto step = [&](auto J) {
            constexpr int j = decltype(J)::value;
            const int c = grp * 4 + j;
            if (c >= W.kc) return;
            const u32x4 w = wc[(long long)c * 64];
            const i32x8 wf = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const u32x4 a = reinterpret_cast<const u32x4 *>(A.codes)[((long long)min(mt + m, A.rt - 1) * A.kc + c) * 64 + lane];
                const i32x8 af = {(int)a[0], (int)a[1], (int)a[2], (int)a[3]};
                acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, af, acc[m], 4, 4, j, sw, j, sa[m]);
            }
        };
        step(std::integral_constant<int, 0>());
        step(std::integral_constant<int, 1>());
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    }
    __shared__ f32x4 part[3][MT][64];
    if (wv) {
#pragma unroll
        for (int m = 0; m < MT; m++) part[wv - 1][m][lane] = acc[m];
    }
    __syncthreads();
    if (wv) return;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        f32x4 v = acc[m];
#pragma unroll
        for (int w = 0; w < 3; w++) v += part[w][m][lane];
        const int row = (mt + m) * 16 + r;
        if (row >= A.rows) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = nt * 16 + 4 * g + j;
            if (n < W.rows) C[row * ldc + n] = (O)v[j];
        }
    }
}

template <class O> static int launch_q(const Mx4View &A, const Mx4View &W, O *C, long long ldc) {
    auto run = [&](auto kernel, int rows, int cols) -> int {   // of row tiles
        const long long mtiles = cdiv(A.rt, rows), ntiles = cdiv(W.rt, cols), wgs = cdiv(mtiles * ntiles, 8) * 8;
        if (wgs > 0xffffff) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm_q: more tiles than one launch can index");
        hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(256), 0, stream, A, W, C, ldc, (int)mtiles, (int)ntiles);
        G9_HIP(hipGetLastError());
        return 0;
    };
    if (A.rt > 4) return cdiv(A.rt, 16) * cdiv(W.rt, 16) >= num_cus ? run(mx4_gemm_q_tile_kernel<O>, 16, 16) : run(mx4_gemm_q_ring_kernel<O>, 8, 8);
    return run(mx4_gemm_q_any_kernel<O>, 4, 1);
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

// Tiles of MT·16 rows × 16·NT·NV columns; k is split until there is about a workgroup a CU.
template <class T, int MT, int NT, int NV, int D> static int launch_few(const Rows &R, const Mx4View &W) {
    const int ntiles = (int)cdiv(W.rt, NT * NV), mtiles = (int)cdiv(R.M, MT * 16);
    const long long tiles = (long long)mtiles * ntiles;
    Split split = {1, nullptr, 0, 0};
    const int ways = (int)(num_cus / tiles), most = W.kc / 4;
    if (ways > 1 && most > 1) {
        split.parts = ways < most ? ways : most;
        G9_TRY(split_space(R, W, &split));
    }
    if (tiles * split.parts > 0x7fffff) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm: more tiles than one launch can index");
    hipLaunchKernelGGL((mx4_gemm_few_kernel<T, T, MT, NT, NV, D, false, false>), dim3((unsigned)(cdiv(tiles * split.parts, 8) * 8)), dim3(NV * 64), 0, stream, R, W, W, 1, mtiles, ntiles, split);
    G9_HIP(hipGetLastError());
    return sum_parts<T>(R, W, split);
}

// Tiles of 64 rows × 256 columns; k is split until there is about a workgroup a CU.
template <class T> static int launch_tiles(const Rows &R, const Mx4View &W) {
    Planes A;
    G9_TRY(stage_planes<T>(R, R.M, W.K, W.kc, &A));
    const int mtiles = (int)cdiv(R.M, 64), ntiles = (int)cdiv(W.rt, 16);
    const long long tiles = (long long)mtiles * ntiles;
    Split split = {1, nullptr, 0, 0};
    const int ways = (int)(num_cus / tiles), most = W.kc / 4;
    if (ways > 1 && most > 1) {
        split.parts = ways < most ? ways : most;
        G9_TRY(split_space(R, W, &split));
    }
    if (tiles * split.parts > 0xffffff) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_gemm: more tiles than one launch can index");
    hipLaunchKernelGGL((mx4_gemm_tile_kernel<T, T, false, false>), dim3((unsigned)(cdiv(tiles * split.parts, 8) * 8)), dim3(256), 0, stream, A, R, W, W, 1, mtiles,
                       ntiles, split);
    G9_HIP(hipGetLastError());
    return sum_parts<T>(R, W, split);
}

template <class T> static int launch_dense(const Rows &R, const Mx4View &W) {
    if (R.M > 64) return launch_tiles<T>(R, W);
    // µs of the product alone, FP16 1 × 11008 × 4096 and FP32 8 × 4096 × 11008: rows kernel 9.4 and 13.2, few kernel 8.8 to
    // 9.5 and 10.7: FP32 rows are taken apart once a workgroup there, and once a wave in the rows kernel.
    if (R.M <= 16) {
        if constexpr (sizeof(T) == 4) return launch_few<T, 1, 2, 8, 4>(R, W);
        else return launch_rows<T>(R, W);
    }
    // 128 columns a workgroup; with 256, which reads the rows from LDS half as often but leaves twice the parts to be summed or half
    // the workgroups: FP32 24 × 4096 × 11008 19.6 µs and 20.0, 24 × 11008 × 4096 21.6 and 20.5, 28 × 2048 × 2048 9.5 and 11.9
    if (R.M <= 32) return launch_few<T, 2, 1, 8, 4>(R, W);
    // FP32 64 × 4096 × 4096 18.6 µs, 56 × 8192 × 8192 40.0, 33 × 1000 × 4992 14.3; 256 columns 21.9, 36.3, 18.1
    return launch_few<T, 4, 1, 8, 2>(R, W);
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
