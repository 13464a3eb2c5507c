// Layer norm over the rows of a matrix (gen9blas_layer_norm) and its gradients (gen9blas_layer_norm_backward).
#include "llm.h"
#include "colsum.h"
#include "rows.h"
#include <algorithm>

namespace g9llm {

// The sum of `v` over the workgroup's 256 threads, in all of them. `part`: four floats that no other sum still uses.
__device__ __forceinline__ float block_sum(float v, float *part) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// y = (x − mean)·rstd·gamma + beta, rstd = 1 / √(mean((x − mean)²) + eps). The mean of x − mean, what rounding has left of it, is
// taken off again: a row whose mean is large against its values loses nothing that x has.
template <class T>
__global__ void __launch_bounds__(256) norm_kernel(const T *__restrict__ X, long long ldx, const float *__restrict__ gamma, const float *__restrict__ beta, float eps, int N,
                                                   T *__restrict__ Y, long long ldy, float *__restrict__ stats) {
    __shared__ float part[3][4];
    const T *x = X + (long long)blockIdx.x * ldx;
    T *y = Y + (long long)blockIdx.x * ldy;
    float s = 0.f;
    for (int n = threadIdx.x; n < N; n += 256) s += (float)x[n];
    const float mean = block_sum(s, part[0]) / N;
    float d = 0.f, q = 0.f;
    for (int n = threadIdx.x; n < N; n += 256) {
        const float v = (float)x[n] - mean;
        d += v, q = __builtin_fmaf(v, v, q);
    }
    const float left = block_sum(d, part[1]) / N, var = block_sum(q, part[2]) / N - left * left, rstd = 1.f / sqrtf(fmaxf(var, 0.f) + eps);
    for (int n = threadIdx.x; n < N; n += 256) {
        const float v = ((float)x[n] - mean - left) * rstd;
        y[n] = (T)(v * (gamma ? gamma[n] : 1.f) + (beta ? beta[n] : 0.f));
    }
    if (stats && threadIdx.x == 0) stats[2LL * blockIdx.x] = mean + left, stats[2LL * blockIdx.x + 1] = rstd;
}

// dx = rstd·(g − mean(g) − x̂·mean(g·x̂)), g = dy·gamma, x̂ = (x − mean)·rstd.
template <class T>
__global__ void __launch_bounds__(256) norm_back_kernel(const T *__restrict__ dY, long long lddy, const T *__restrict__ X, long long ldx, const float *__restrict__ stats,
                                                        const float *__restrict__ gamma, int N, T *__restrict__ dX, long long lddx) {
    __shared__ float part[2][4];
    const T *x = X + (long long)blockIdx.x * ldx, *dy = dY + (long long)blockIdx.x * lddy;
    T *dx = dX + (long long)blockIdx.x * lddx;
    const float mean = stats[2LL * blockIdx.x], rstd = stats[2LL * blockIdx.x + 1];
    float a = 0.f, b = 0.f;
    for (int n = threadIdx.x; n < N; n += 256) {
        const float g = (float)dy[n] * (gamma ? gamma[n] : 1.f);
        a += g, b = __builtin_fmaf(g, ((float)x[n] - mean) * rstd, b);
    }
    a = block_sum(a, part[0]) / N, b = block_sum(b, part[1]) / N;
    for (int n = threadIdx.x; n < N; n += 256) {
        const float g = (float)dy[n] * (gamma ? gamma[n] : 1.f);
        dx[n] = (T)(rstd * (g - a - ((float)x[n] - mean) * rstd * b));
    }
}

// Sums of dy·x̂ and of dy over blocks of rows: part 2b and 2b + 1 of N.
template <class T>
__global__ void __launch_bounds__(256) norm_sums_kernel(const T *__restrict__ dY, long long lddy, const T *__restrict__ X, long long ldx, const float *__restrict__ stats,
                                                        int M, int N, int rows, float *__restrict__ sums) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    const long long m0 = (long long)blockIdx.y * rows, m1 = min(m0 + rows, (long long)M);
    float a = 0.f, b = 0.f;
    for (long long m = m0; m < m1; m++) {
        const float g = (float)dY[m * lddy + n];
        a = __builtin_fmaf(g, ((float)X[m * ldx + n] - stats[2 * m]) * stats[2 * m + 1], a), b += g;
    }
    sums[2LL * blockIdx.y * N + n] = a;
    sums[(2LL * blockIdx.y + 1) * N + n] = b;
}

template <class T>
static int norm(int M, int N, const T *X, int ldx, const float *gamma, const float *beta, float eps, T *Y, int ldy, float *stats) {
    return by_rows(M, 256, [&](long long m0, unsigned rows) -> int {
        hipLaunchKernelGGL((norm_kernel<T>), dim3(rows), dim3(256), 0, stream, X + m0 * ldx, ldx, gamma, beta, eps, N, Y + m0 * ldy, ldy, stats ? stats + 2 * m0 : nullptr);
        G9_HIP(hipGetLastError());
        return 0;
    });
}
template <class T>
static int norm_back(int M, int N, const T *dY, int lddy, const T *X, int ldx, const float *stats, const float *gamma, T *dX, int lddx, float *dgamma, float *dbeta, int accumulate) {
    if (dX)
        G9_TRY(by_rows(M, 256, [&](long long m0, unsigned rows) -> int {
            hipLaunchKernelGGL((norm_back_kernel<T>), dim3(rows), dim3(256), 0, stream, dY + m0 * lddy, lddy, X + m0 * ldx, ldx, stats + 2 * m0, gamma, N, dX + m0 * lddx, lddx);
            G9_HIP(hipGetLastError());
            return 0;
        }));
    if (dgamma || dbeta) {
        const int rows = (int)std::max(32LL, cdiv(M, 512));
        const long long blocks = cdiv(M, rows);
        void *sums;
        G9_TRY(scratch(SLOT_SUMS, (size_t)blocks * 2 * N * 4, &sums));
        hipLaunchKernelGGL((norm_sums_kernel<T>), dim3((unsigned)cdiv(N, 256), (unsigned)blocks), dim3(256), 0, stream, dY, lddy, X, ldx, stats, M, N, rows, (float *)sums);
        G9_HIP(hipGetLastError());
        if (dgamma) G9_TRY(column_sums((float *)sums, blocks, N, 2LL * N, dgamma, accumulate));
        if (dbeta) G9_TRY(column_sums((float *)sums + N, blocks, N, 2LL * N, dbeta, accumulate));
    }
    return 0;
}

}  // namespace g9llm

using namespace g9llm;

extern "C" {

int gen9blas_layer_norm(int type, int M, int N, const void *X, int ldx, const float *gamma, const float *beta, float eps, void *Y, int ldy, float *stats) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "layer_norm: type %d unavailable", type);
    if (M <= 0) return 0;
    if (N < 1 || ldx < N || ldy < N || !(eps >= 0)) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "layer_norm: N %d, ldx %d, ldy %d, eps %g", N, ldx, ldy, eps);
    const size_t es = elem_size(type);
    G9_TRY(need_device(X, ((size_t)(M - 1) * ldx + N) * es, "layer_norm: X"));
    if (gamma) G9_TRY(need_device(gamma, (size_t)N * 4, "layer_norm: gamma"));
    if (beta) G9_TRY(need_device(beta, (size_t)N * 4, "layer_norm: beta"));
    G9_TRY(need_device(Y, ((size_t)(M - 1) * ldy + N) * es, "layer_norm: Y"));
    if (stats) G9_TRY(need_device(stats, (size_t)M * 8, "layer_norm: stats"));
    return type == GEN9BLAS_H ? norm(M, N, (const _Float16 *)X, ldx, gamma, beta, eps, (_Float16 *)Y, ldy, stats) : norm(M, N, (const float *)X, ldx, gamma, beta, eps, (float *)Y, ldy, stats);
}

int gen9blas_layer_norm_backward(int type, int M, int N, const void *dY, int lddy, const void *X, int ldx, const float *stats, const float *gamma, void *dX, int lddx,
                                 float *dgamma, float *dbeta, int accumulate) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "layer_norm_backward: type %d unavailable", type);
    if (!dX && !dgamma && !dbeta) return 0;
    M = std::max(M, 0);
    if (N < 1 || lddy < N || ldx < N || (dX && lddx < N)) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "layer_norm_backward: N %d, lddy %d, ldx %d, lddx %d", N, lddy, ldx, lddx);
    const size_t es = elem_size(type);
    if (M) {
        G9_TRY(need_device(dY, ((size_t)(M - 1) * lddy + N) * es, "layer_norm_backward: dY"));
        G9_TRY(need_device(X, ((size_t)(M - 1) * ldx + N) * es, "layer_norm_backward: X"));
        G9_TRY(need_device(stats, (size_t)M * 8, "layer_norm_backward: stats"));
        if (dX) G9_TRY(need_device(dX, ((size_t)(M - 1) * lddx + N) * es, "layer_norm_backward: dX"));
    }
    if (gamma) G9_TRY(need_device(gamma, (size_t)N * 4, "layer_norm_backward: gamma"));
    if (dgamma) G9_TRY(need_device(dgamma, (size_t)N * 4, "layer_norm_backward: dgamma"));
    if (dbeta) G9_TRY(need_device(dbeta, (size_t)N * 4, "layer_norm_backward: dbeta"));
    if (!M) {   // sums over no rows
        if (accumulate) return 0;
        if (dgamma) G9_TRY(zero_rows(dgamma, 4LL * N, 1, 4LL * N));
        return dbeta ? zero_rows(dbeta, 4LL * N, 1, 4LL * N) : 0;
    }
    return type == GEN9BLAS_H ? norm_back(M, N, (const _Float16 *)dY, lddy, (const _Float16 *)X, ldx, stats, gamma, (_Float16 *)dX, lddx, dgamma, dbeta, accumulate)
                              : norm_back(M, N, (const float *)dY, lddy, (const float *)X, ldx, stats, gamma, (float *)dX, lddx, dgamma, dbeta, accumulate);
}

}  // extern "C"
