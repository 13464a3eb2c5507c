// Products with MX4 weights on the matrix cores: fragments, and the kernel that takes every shape.
#pragma once
#include "llm.h"
#include "lds_dma.h"

namespace g9llm {

// How activations of type T meet 4-bit weights, eight k per lane and MFMA.
// FP16: FP16 weights scaled by the row's exponent (one product). FP32: BF16 weights, which hold any code and scale
// exactly, times the activation in three BF16 pieces of 8 bits each, a = a1 + a2 + a3 exactly (by truncation; below
// 2^-110 the last bits underflow): FP32 products from three BF16 ones, at three times their cost instead of the sixteen
// of the FP32 matrix cores.
template <class T> struct Act;
template <> struct Act<_Float16> {
    static constexpr int P = 1;
    typedef f16x8 Frag;
    // 8 codes of a word to FP16, scale byte s of a block of a row whose largest is e
    static __device__ __forceinline__ float scale(unsigned s, int e) {
        const int r = s == 255 ? 255 : max((int)s - e + 140, 0);
        return __builtin_bit_cast(float, r << 23);
    }
    static __device__ __forceinline__ Frag weights(unsigned w, float scale) {
        const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1);
        const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3);
        return Frag{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    static __device__ __forceinline__ void split(const _Float16 *v, Frag *f) { __builtin_memcpy(f, v, 16); }
    static __device__ __forceinline__ f32x4 mfma(Frag w, Frag a, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(w, a, c, 0, 0, 0); }
    static __device__ __forceinline__ float finish(float v, int e) { return ldexpf(v, e - 140); }
};
template <> struct Act<float> {
    static constexpr int P = 3;
    typedef bf16x8 Frag;
    static __device__ __forceinline__ float scale(unsigned s, int) { return __builtin_bit_cast(float, s << 23); }
    static __device__ __forceinline__ Frag weights(unsigned w, float scale) {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
        const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
        return Frag{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    // An infinity is all in the first piece; a NaN whose payload lies in the low bits stays a NaN.
    static __device__ __forceinline__ void split(const float *v, Frag *f) {
        unsigned p[3][8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const unsigned u = __builtin_bit_cast(unsigned, v[i]);
            const bool finite = (u & 0x7f800000u) != 0x7f800000u;
            p[0][i] = finite || !(u & 0x7fffffu) ? u & 0xffff0000u : 0x7fc00000u;
            const float r = finite ? v[i] - __builtin_bit_cast(float, p[0][i]) : 0.f;
            p[1][i] = __builtin_bit_cast(unsigned, r) & 0xffff0000u;
            p[2][i] = __builtin_bit_cast(unsigned, r - __builtin_bit_cast(float, p[1][i]));
        }
#pragma unroll
        for (int q = 0; q < 3; q++) {
            u32x4 o;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = p[q][2 * i] >> 16 | (p[q][2 * i + 1] & 0xffff0000u);
            f[q] = __builtin_bit_cast(Frag, o);
        }
    }
    static __device__ __forceinline__ f32x4 mfma(Frag w, Frag a, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, a, c, 0, 0, 0); }
    static __device__ __forceinline__ float finish(float v, int) { return v; }
};

// The largest scale byte of a row of W.
__device__ __forceinline__ int row_top(const uint8_t *top, int kt) {
    unsigned m = 0;
    for (int i = 0; i < kt; i += 4) {
        const unsigned w = *reinterpret_cast<const unsigned *>(top + i);
        m = max(max(m, max(w & 255u, w >> 8 & 255u)), max(w >> 16 & 255u, w >> 24));
    }
    return (int)m;
}

// 8 consecutive elements of a row, zeros past K.
template <class T> __device__ __forceinline__ void load8(const T *row, int k, int K, T *v) {
    constexpr int V = 16 / sizeof(T);
    if (k + 8 <= K) {
#pragma unroll
        for (int i = 0; i < 8 / V; i++) {
            const g9::dma_u32x4 q = g9::load16u(row + k + i * V);
            __builtin_memcpy(v + i * V, &q, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = k + i < K ? row[k + i] : T(0);
    }
}

// Rows of a product: dense (row m at A + m·ldt, result at C + m·ldct), or of the experts: a list of tiles (expert, first
// place in `order`), `order` the slots t·S + s by expert, off[e] where expert e's begin.
struct Rows {
    const void *A;
    void *C;
    long long ldt, lds, ldct, ldcs;
    int M, S;
    const int *tiles, *order, *off;
};

__device__ __forceinline__ float silu(float z) { return z / (1.f + expf(-z)); }

// The product of any shape. A workgroup makes MT·16 rows × 16 columns, its 4 waves every fourth tile of k, summed in wave
// order through LDS. Weights are the first operand: lane 16g + r holds columns n = 4g .. 4g+3 of activation row r.
template <class T, class O, int MT, bool GROUPED, bool GATED>
__global__ void __launch_bounds__(256) mx4_gemm_any_kernel(Rows R, Mx4View W, Mx4View G, int experts) {
    typedef Act<T> X;
    typedef typename X::Frag Frag;
    constexpr int NW = GATED ? 2 : 1;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int nt = blockIdx.x % W.rt;
    const int mt = blockIdx.x / W.rt;
    int first, count, e = 0;   // rows first .. first + count − 1 (dense), or places in `order`
    if (GROUPED) {
        e = R.tiles[2 * mt];
        if (e < 0) return;   // past the last tile
        first = R.tiles[2 * mt + 1];
        count = min(MT * 16, R.off[e + 1] - first);
    } else {
        first = mt * MT * 16;
        count = min(MT * 16, R.M - first);
    }
    const T *arow[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int i = m * 16 + r;
        if (i >= count) arow[m] = nullptr;
        else if (GROUPED) {
            const int slot = R.order[first + i];
            arow[m] = (const T *)R.A + (slot / R.S) * R.ldt + (slot % R.S) * R.lds;
        } else
            arow[m] = (const T *)R.A + (long long)(first + i) * R.ldt;
    }
    f32x4 acc[NW][MT];
#pragma unroll
    for (int q = 0; q < NW; q++)
#pragma unroll
        for (int m = 0; m < MT; m++) acc[q][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    int top[NW];
    if (!GROUPED || e < experts) {
        const long long tile = (long long)e * W.rt + nt;
#pragma unroll
        for (int q = 0; q < NW; q++) top[q] = row_top((q ? G.top : W.top) + (tile * 16 + r) * W.kt, W.kt);
        for (int c = wv; c < W.kc; c += 4) {
            u32x4 w[NW];
            float sc[NW];
#pragma unroll
            for (int q = 0; q < NW; q++) {
                w[q] = reinterpret_cast<const u32x4 *>(q ? G.codes : W.codes)[(tile * W.kc + c) * 64 + lane];
                sc[q] = X::scale((q ? G.scales : W.scales)[(tile * W.kg + c / 4) * 256 + lane * 4 + c % 4], top[q]);
            }
            Frag a[MT][4][X::P];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    T v[8];
                    if (arow[m]) load8(arow[m], c * 128 + g * 32 + i * 8, W.K, v);
                    else
#pragma unroll
                        for (int j = 0; j < 8; j++) v[j] = T(0);
                    X::split(v, a[m][i]);
                }
#pragma unroll
            for (int q = 0; q < NW; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const Frag wf = X::weights(w[q][i], sc[q]);
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int p = X::P - 1; p >= 0; p--) acc[q][m] = X::mfma(wf, a[m][i][p], acc[q][m]);
                }
        }
    } else {
#pragma unroll
        for (int q = 0; q < NW; q++) top[q] = 0;   // empty places: zeros
    }
    __shared__ f32x4 part[3][NW * MT][64];
    if (wv) {
#pragma unroll
        for (int q = 0; q < NW; q++)
#pragma unroll
            for (int m = 0; m < MT; m++) part[wv - 1][q * MT + m][lane] = acc[q][m];
    }
    __syncthreads();
    if (wv) return;
    int tn[NW][4];
#pragma unroll
    for (int q = 0; q < NW; q++)
#pragma unroll
        for (int j = 0; j < 4; j++) tn[q][j] = __shfl(top[q], 4 * g + j);
#pragma unroll
    for (int m = 0; m < MT; m++) {
        float y[NW][4];
#pragma unroll
        for (int q = 0; q < NW; q++) {
            f32x4 v = acc[q][m];
#pragma unroll
            for (int w = 0; w < 3; w++) v += part[w][q * MT + m][lane];
#pragma unroll
            for (int j = 0; j < 4; j++) y[q][j] = X::finish(v[j], tn[q][j]);
        }
        const int i = m * 16 + r;
        if (i >= count) continue;
        O *c;
        if (GROUPED) {
            const int slot = R.order[first + i];
            c = (O *)R.C + (slot / R.S) * R.ldct + (slot % R.S) * R.ldcs;
        } else
            c = (O *)R.C + (long long)(first + i) * R.ldct;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = nt * 16 + 4 * g + j;
            if (n < W.rows) c[n] = (O)(GATED ? silu(y[NW - 1][j]) * y[0][j] : y[0][j]);
        }
    }
}

}  // namespace g9llm
