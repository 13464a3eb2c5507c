// MX4 matrices: creation, quantisation, loading of a checkpoint's rows, and the values back.
#include "llm.h"
#include "lds_dma.h"
#include <new>

namespace g9llm {

// 32 consecutive elements of a row from k on, zeros past K. Whole blocks in 16-byte loads at element alignment.
template <class T> __device__ __forceinline__ void load32(const T *__restrict__ row, long long k, int K, T *v) {
    constexpr int V = 16 / sizeof(T);
    if (k + 32 <= K) {
#pragma unroll
        for (int i = 0; i < 32 / V; i++) {
            const g9::dma_u32x4 q = g9::load16u(row + k + i * V);
            __builtin_memcpy(v + i * V, &q, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = k + i < K ? row[k + i] : T(0);
    }
}

// One block to its scale byte and codes. The exponent field of the largest magnitude in FP32 is ⌊log2⌋ + 127; the scale is
// two below, so that the largest becomes 4..8 (beyond 6: 6). v_cvt_scalef32_pk_fp4_f32 divides by the scale, rounds to
// nearest with ties to the even code, and saturates.
template <class T> __device__ __forceinline__ unsigned quantize32(const T *v, u32x4 &codes) {
    float m = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        const float a = __builtin_fabsf((float)v[i]);
        bad |= !(a < __builtin_inff());
        m = fmaxf(m, a);
    }
    const unsigned field = __builtin_bit_cast(unsigned, m) >> 23;
    const unsigned s = bad ? 255u : (unsigned)max((int)field - 2, 0);
    const float scale = __builtin_bit_cast(float, s << 23);
#pragma unroll
    for (int w = 0; w < 4; w++) {
        unsigned c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, (float)v[8 * w], (float)v[8 * w + 1], scale, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, (float)v[8 * w + 2], (float)v[8 * w + 3], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, (float)v[8 * w + 4], (float)v[8 * w + 5], scale, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, (float)v[8 * w + 6], (float)v[8 * w + 7], scale, 3);
        codes[w] = bad ? 0u : c;
    }
    return s;
}

// Scale bytes of a row tile's 512-k group: sc[j] of wave j's lanes, written as one word per lane with the row's largest.
__device__ __forceinline__ void write_scales(unsigned char (*sc)[64], uint8_t *scales, uint8_t *top, int kt, int grp) {
    __syncthreads();
    const int t = threadIdx.x;
    if (t < 64) {
        const unsigned w = sc[0][t] | sc[1][t] << 8 | sc[2][t] << 16 | (unsigned)sc[3][t] << 24;
        reinterpret_cast<unsigned *>(scales)[t] = w;
        int m = max(max(sc[0][t], sc[1][t]), max(sc[2][t], sc[3][t]));
        m = max(m, __shfl_xor(m, 16));
        m = max(m, __shfl_xor(m, 32));
        if (t < 16) top[t * kt + grp] = (uint8_t)m;
    }
}

// A workgroup makes one row tile's group of 512 k, wave j its tile j: lane 16g + r the block of row r, k = 32g. HBM bounds it:
// 11008 × 4096 FP32 43 µs, 4.7 TB/s.
template <class T>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(const T *__restrict__ X, long long ldx, long long sX, Mx4View q,
                                                           uint8_t *codes, uint8_t *scales, uint8_t *top) {
    __shared__ unsigned char sc[4][64];
    const int lane = threadIdx.x & 63, j = threadIdx.x >> 6;
    const int grp = blockIdx.x % q.kg;
    const long long tile = blockIdx.x / q.kg;   // over all matrices
    const int b = (int)(tile / q.rt), row = (int)(tile % q.rt) * 16 + (lane & 15), c = grp * 4 + j;
    unsigned s = 0;
    if (c < q.kc) {
        const long long k = (long long)c * 128 + (lane >> 4) * 32;
        u32x4 w = {0, 0, 0, 0};
        if (row < q.rows && k < q.K) {
            T v[32];
            load32(X + b * sX + row * ldx, k, q.K, v);
            s = quantize32(v, w);   // of a block of zeros: 0, as every other scale leaves the largest at 4 or more
        }
        reinterpret_cast<u32x4 *>(codes)[(tile * q.kc + c) * 64 + lane] = w;
    }
    sc[j][lane] = (unsigned char)s;
    write_scales(sc, scales + (tile * q.kg + grp) * 256, top + tile * 16 * q.kt, q.kt, grp);
}

// The same from a checkpoint's rows of codes and scales. Codes past K are cleared; a block of zeros, which may come with any
// scale, gets scale 0 (NaN blocks, 255, stay).
__global__ void __launch_bounds__(256) mx4_load_kernel(const uint8_t *__restrict__ in, long long ldc, const uint8_t *__restrict__ sin,
                                                       long long lds, Mx4View q, uint8_t *codes, uint8_t *scales, uint8_t *top) {
    __shared__ unsigned char sc[4][64];
    const int lane = threadIdx.x & 63, j = threadIdx.x >> 6;
    const int grp = blockIdx.x % q.kg;
    const long long tile = blockIdx.x / q.kg;
    const int b = (int)(tile / q.rt), row = (int)(tile % q.rt) * 16 + (lane & 15), c = grp * 4 + j;
    unsigned s = 0;
    if (c < q.kc) {
        const int k = c * 128 + (lane >> 4) * 32;
        union { u32x4 v; uint8_t e[16]; } w;
        w.v = u32x4{0, 0, 0, 0};
        if (row < q.rows && k < q.K) {
            const uint8_t *p = in + ((long long)b * q.rows + row) * ldc + k / 2;
            s = sin[((long long)b * q.rows + row) * lds + k / 32];
            if (k + 32 <= q.K) {
                const g9::dma_u32x4 d = g9::load16u(p);
                w.v = u32x4{d[0], d[1], d[2], d[3]};
            } else {
                const int n = q.K - k;
#pragma unroll
                for (int i = 0; i < 16; i++) w.e[i] = 2 * i + 1 < n ? p[i] : 2 * i < n ? p[i] & 15 : 0;
            }
            if (!((w.v[0] | w.v[1] | w.v[2] | w.v[3]) & 0x77777777u) && s != 255) s = 0;
        }
        reinterpret_cast<u32x4 *>(codes)[(tile * q.kc + c) * 64 + lane] = w.v;
    }
    sc[j][lane] = (unsigned char)s;
    write_scales(sc, scales + (tile * q.kg + grp) * 256, top + tile * 16 * q.kt, q.kt, grp);
}

// A wave's tile of 16 rows × 128 k: the codes through LDS, so that 32 lanes write 512 consecutive bytes of a row, four values
// each (11008 × 4096 30 µs, 6.8 TB/s into HBM and the last cache; a lane that wrote its block's 128 bytes 54).
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(Mx4View q, float *__restrict__ X, long long ldx, long long sX) {
    __shared__ u32x4 codes[4][64];
    __shared__ unsigned char sc[4][64];
    const int lane = threadIdx.x & 63, j = threadIdx.x >> 6;
    const int grp = blockIdx.x % q.kg;
    const long long tile = blockIdx.x / q.kg;
    const int b = (int)(tile / q.rt), row0 = (int)(tile % q.rt) * 16, c = grp * 4 + j;
    if (c < q.kc) {
        codes[j][lane] = reinterpret_cast<const u32x4 *>(q.codes)[(tile * q.kc + c) * 64 + lane];
        sc[j][lane] = q.scales[(tile * q.kg + grp) * 256 + lane * 4 + j];
    }
    __syncthreads();
    const int l = lane & 31, g = l >> 3, k = c * 128 + l * 4;
    if (c >= q.kc || k >= q.K) return;
    float *x = X + b * sX + k;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = 2 * i + (lane >> 5);
        if (row0 + r >= q.rows) continue;
        const unsigned w = reinterpret_cast<const unsigned short *>(&codes[j][16 * g + r])[l & 7];
        const float scale = __builtin_bit_cast(float, (unsigned)sc[j][16 * g + r] << 23);
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
        float *at = x + (row0 + r) * ldx;
        if (k + 4 <= q.K) {
            typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
            *reinterpret_cast<F4 *>(at) = F4{a[0], a[1], e[0], e[1]};
        } else {
            const float v[4] = {a[0], a[1], e[0], e[1]};
#pragma unroll
            for (int n = 0; n < 4; n++)
                if (k + n < q.K) at[n] = v[n];
        }
    }
}

static size_t span(long long count, long long stride, long long rows, long long ld, long long cols) {
    return (size_t)((count - 1) * stride + (rows - 1) * ld + cols);
}

}  // namespace g9llm

using namespace g9llm;

extern "C" {

gen9blas_mx4 *gen9blas_mx4_create(int count, int rows, int K) {
    if (begin()) return nullptr;
    if (count < 1 || rows < 1 || K < 1) {
        fail(GEN9BLAS_ERR_INVALID_ARG, "mx4_create: count = %d, rows = %d, K = %d", count, rows, K);
        return nullptr;
    }
    if (K > MAX_COLS) {
        fail(GEN9BLAS_ERR_UNSUPPORTED, "mx4_create: K = %d, rows have at most %d values", K, MAX_COLS);
        return nullptr;
    }
    gen9blas_mx4 q;
    q.count = count, q.rows = rows, q.K = K;
    q.rt = (int)cdiv(rows, 16), q.kc = (int)cdiv(K, 128), q.kg = (int)cdiv(q.kc, 4), q.kt = (int)cdiv(q.kg, 16) * 16;
    const long long tiles = (long long)count * q.rt;
    if (tiles * q.kg > 0xffffffLL) {
        fail(GEN9BLAS_ERR_UNSUPPORTED, "mx4_create: %d × %d × %d is more than one launch can index", count, rows, K);
        return nullptr;
    }
    const size_t nc = (size_t)tiles * q.kc * 1024, ns = (size_t)tiles * q.kg * 256, nt = (size_t)tiles * 16 * q.kt;
    void *buf = nullptr;
    const hipError_t e = hipMalloc(&buf, nc + ns + nt);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        fail(GEN9BLAS_ERR_OUT_OF_MEMORY, "mx4_create: hipMalloc(%zu): %s", nc + ns + nt, hipGetErrorString(e));
        return nullptr;
    }
    q.codes = (uint8_t *)buf, q.scales = q.codes + nc, q.top = q.scales + ns;
    gen9blas_mx4 *Q = new (std::nothrow) gen9blas_mx4(q);
    hipError_t ke = Q ? hipMemsetAsync(buf, 0, nc + ns + nt, stream) : hipSuccess;
    if (!Q || ke != hipSuccess) {
        (void)hipFree(buf);
        delete Q;
        if (ke != hipSuccess) hip_fail(ke, "mx4_create", __FILE__, __LINE__);
        else fail(GEN9BLAS_ERR_OUT_OF_MEMORY, "mx4_create: out of host memory");
        return nullptr;
    }
    return Q;
}

void gen9blas_mx4_free(gen9blas_mx4 *Q) {
    if (!Q || begin()) return;
    (void)hipStreamSynchronize(stream);   // queued products may still read it
    (void)hipFree(Q->codes);
    delete Q;
}

int gen9blas_mx4_quantize(int type, const void *X, int ldx, int64_t sX, gen9blas_mx4 *Q) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "mx4_quantize: type %d unavailable", type);
    if (!Q) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_quantize: no matrix");
    if (ldx < Q->K || (Q->count > 1 && sX < 0)) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_quantize: ldx %d < K %d, or a negative stride", ldx, Q->K);
    G9_TRY(need_device(X, span(Q->count, sX, Q->rows, ldx, Q->K) * elem_size(type), "mx4_quantize: X"));
    const dim3 grid((unsigned)((long long)Q->count * Q->rt * Q->kg)), block(256);
    if (type == GEN9BLAS_H)
        hipLaunchKernelGGL((mx4_quantize_kernel<_Float16>), grid, block, 0, stream, (const _Float16 *)X, (long long)ldx, (long long)sX,
                           view(Q), Q->codes, Q->scales, Q->top);
    else
        hipLaunchKernelGGL((mx4_quantize_kernel<float>), grid, block, 0, stream, (const float *)X, (long long)ldx, (long long)sX, view(Q),
                           Q->codes, Q->scales, Q->top);
    G9_HIP(hipGetLastError());
    return 0;
}

int gen9blas_mx4_load(const uint8_t *codes, int ldc, const uint8_t *scales, int lds, gen9blas_mx4 *Q) {
    G9_TRY(begin());
    if (!Q) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_load: no matrix");
    const int nc = (int)cdiv(Q->K, 2), ns = (int)cdiv(Q->K, 32);
    if (ldc < nc || lds < ns) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_load: ldc %d < %d or lds %d < %d", ldc, nc, lds, ns);
    const long long rows = (long long)Q->count * Q->rows;
    G9_TRY(need_device(codes, span(1, 0, rows, ldc, nc), "mx4_load: codes"));
    G9_TRY(need_device(scales, span(1, 0, rows, lds, ns), "mx4_load: scales"));
    hipLaunchKernelGGL(mx4_load_kernel, dim3((unsigned)((long long)Q->count * Q->rt * Q->kg)), dim3(256), 0, stream, codes, (long long)ldc,
                       scales, (long long)lds, view(Q), Q->codes, Q->scales, Q->top);
    G9_HIP(hipGetLastError());
    return 0;
}

int gen9blas_mx4_dequantize(const gen9blas_mx4 *Q, float *X, int ldx, int64_t sX) {
    G9_TRY(begin());
    if (!Q) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_dequantize: no matrix");
    if (ldx < Q->K || (Q->count > 1 && sX < (int64_t)(Q->rows - 1) * ldx + Q->K))
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "mx4_dequantize: ldx %d < K %d, or matrices that overlap", ldx, Q->K);
    G9_TRY(need_device(X, span(Q->count, sX, Q->rows, ldx, Q->K) * 4, "mx4_dequantize: X"));
    hipLaunchKernelGGL(mx4_dequantize_kernel, dim3((unsigned)((long long)Q->count * Q->rt * Q->kg)), dim3(256), 0, stream, view(Q), X,
                       (long long)ldx, (long long)sX);
    G9_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
