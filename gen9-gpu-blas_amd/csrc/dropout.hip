// gen9blas_dropout: Y = dropout(X) + R.
#include "llm.h"
#include "dropout.h"
#include "rows.h"

namespace g9llm {

// A thread has the eight columns of a Philox counter. The mask is made where it is used and never stored. HBM bounds it: 8192 × 11008
// FP16 with R 96 µs, 541 MB at 5.6 TB/s (Philox's 20 products of 32 bits for 8 elements run beside the loads).
template <class T>
__global__ void __launch_bounds__(256) dropout_kernel(const T *__restrict__ X, long long ldx, Dropout d, const T *__restrict__ R, long long ldr, int M, int N, int groups,
                                                      T *__restrict__ Y, long long ldy) {
    const long long total = (long long)M * groups;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long m = i / groups;
        const int n = (int)(i % groups) * 8, valid = N - n;
        float v[8];
        load_some<8>(X + m * ldx + n, valid, v);
        drop<8>(d, (unsigned)m, n, v);
        if (R) {
            float r[8];
            load_some<8>(R + m * ldr + n, valid, r);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += r[e];
        }
        store_some<8>(Y + m * ldy + n, valid, v);
    }
}

template <class T> static int dropout(int M, int N, const T *X, int ldx, const Dropout &d, const T *R, int ldr, T *Y, int ldy) {
    const int groups = (int)cdiv(N, 8);
    const long long wgs = cdiv((long long)M * groups, 256);
    hipLaunchKernelGGL((dropout_kernel<T>), dim3((unsigned)std::min(wgs, 16LL << 10)), dim3(256), 0, stream, X, ldx, d, R, ldr, M, N, groups, Y, ldy);
    G9_HIP(hipGetLastError());
    return 0;
}

}  // namespace g9llm

using namespace g9llm;

extern "C" int gen9blas_dropout(int type, int M, int N, const void *X, int ldx, double p, uint64_t seed, uint64_t offset, const void *R, int ldr, void *Y, int ldy) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "dropout: type %d unavailable", type);
    if (!(p >= 0 && p <= 1)) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "dropout: %g is not in [0, 1]", p);
    if (M <= 0 || N <= 0) return 0;
    if (ldx < N || ldy < N || (R && ldr < N)) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "dropout: N %d, ldx %d, ldr %d, ldy %d", N, ldx, ldr, ldy);
    const size_t es = elem_size(type);
    G9_TRY(need_device(X, ((size_t)(M - 1) * ldx + N) * es, "dropout: X"));
    if (R) G9_TRY(need_device(R, ((size_t)(M - 1) * ldr + N) * es, "dropout: R"));
    G9_TRY(need_device(Y, ((size_t)(M - 1) * ldy + N) * es, "dropout: Y"));
    const Dropout d = make_dropout(p, seed, offset);
    return type == GEN9BLAS_H ? dropout(M, N, (const _Float16 *)X, ldx, d, (const _Float16 *)R, ldr, (_Float16 *)Y, ldy)
                              : dropout(M, N, (const float *)X, ldx, d, (const float *)R, ldr, (float *)Y, ldy);
}
