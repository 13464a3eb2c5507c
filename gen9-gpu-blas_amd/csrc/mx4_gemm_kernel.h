// Products of FP16 and FP32 rows with MX4 weights: what their kernels share.
#pragma once
#include "llm.h"
#include "lds_dma.h"
#include <type_traits>

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
    // 8 codes of a word to FP16, scale byte s of a block of a row whose largest is e: s <= e, or s = 255, which makes every
    // code a NaN, zeros too
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
    // U elements of a row, as each plane has them
    template <int U> using Piece = typename std::conditional<U == 8, u32x4, unsigned long long>::type;
    template <int U, class V> static __device__ __forceinline__ void split_unit(V v, Piece<U> *h) { __builtin_memcpy(h, &v, U * 2); }
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
    // The pieces of two elements, each in the halves of a word. An infinity is all in the first piece; a NaN whose payload
    // lies in the low bits stays a NaN.
    static __device__ __forceinline__ void split2(float x, float y, unsigned *h) {
        unsigned p[3][2];
        const float v[2] = {x, y};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const unsigned u = __builtin_bit_cast(unsigned, v[i]);
            const bool finite = (u & 0x7f800000u) != 0x7f800000u;
            p[0][i] = finite || !(u & 0x7fffffu) ? u : 0x7fc00000u;
            const float r = finite ? v[i] - __builtin_bit_cast(float, u & 0xffff0000u) : 0.f;
            p[1][i] = __builtin_bit_cast(unsigned, r);
            p[2][i] = __builtin_bit_cast(unsigned, r - __builtin_bit_cast(float, p[1][i] & 0xffff0000u));
        }
#pragma unroll
        for (int q = 0; q < 3; q++) h[q] = __builtin_amdgcn_perm(p[q][1], p[q][0], 0x07060302u);   // the high halves
    }
    static __device__ __forceinline__ void split(const float *v, Frag *f) {
        u32x4 o[3];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            unsigned h[3];
            split2(v[2 * i], v[2 * i + 1], h);
            o[0][i] = h[0], o[1][i] = h[1], o[2][i] = h[2];
        }
#pragma unroll
        for (int q = 0; q < 3; q++) f[q] = __builtin_bit_cast(Frag, o[q]);
    }
    template <int U> using Piece = unsigned long long;
    template <int U, class V> static __device__ __forceinline__ void split_unit(V v, unsigned long long *h) {
        static_assert(U == 4, "one 16-byte load");
        unsigned a[3], b[3];
        split2(v[0], v[1], a);
        split2(v[2], v[3], b);
#pragma unroll
        for (int q = 0; q < 3; q++) h[q] = (unsigned long long)b[q] << 32 | a[q];
    }
    static __device__ __forceinline__ f32x4 mfma(Frag w, Frag a, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, a, c, 0, 0, 0); }
    static __device__ __forceinline__ float finish(float v, int) { return v; }
};

// The largest scale bytes of N rows of W, top[n] .. top[n] + kt − 1 (kt: a multiple of 16): the loads of all rows together.
template <int N> __device__ __forceinline__ void row_tops(const uint8_t *const *top, int kt, int *out) {
    u32x4 v[N];
#pragma unroll
    for (int n = 0; n < N; n++) v[n] = *reinterpret_cast<const u32x4 *>(top[n]), out[n] = 0;
    for (int i = 0; i < kt; i += 16) {
        u32x4 next[N];
#pragma unroll
        for (int n = 0; n < N; n++) next[n] = *reinterpret_cast<const u32x4 *>(top[n] + min(i + 16, kt - 16));
#pragma unroll
        for (int n = 0; n < N; n++) {
            unsigned m = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) m = max(max(m, max(v[n][j] & 255u, v[n][j] >> 8 & 255u)), max(v[n][j] >> 16 & 255u, v[n][j] >> 24));
            out[n] = max(out[n], (int)m);
            v[n] = next[n];
        }
    }
}

// Rows of 128 k in LDS (256 bytes of FP16 or BF16): 16-byte piece q of row m lies at q ^ swizzle(m). ds_read_b128 takes lanes
// 0-3, 12-15 and 20-27 together (and 4-11, 16-19 and 28-31): rows of two pieces that differ in bit 2. With the rows 0-3 and
// 12-15 at 0..7 and the others at 8..15 these sixteen lie in different banks; q ^ (m & 15) had them in pairs (half of the LDS
// cycles of 1000 × 11008 × 4096).
__device__ __forceinline__ int swizzle(int m) { return (m & 3) | (m >> 1 & 4) | ((m >> 3 ^ m >> 2) & 1) << 3; }

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
    const int *ids;   // not null: no plan, M places with these experts
};

// Rows of a finished tile from LDS (ROWS rows of COLS elements, PITCH bytes apart) to memory: consecutive threads take
// consecutive 16 bytes of a row, so that whole lines are written. As the matrix cores leave it a tile would go out in pieces of 16 and
// 32 bytes: 4096 × 11008 × 512 of two MX4 matrices 48 µs, 37 of them outside the products.
// row(i): where row i of the tile begins, or null; n: columns from there that exist.
template <class O, int NTH, int ROWS, int COLS, int PITCH, class F>
__device__ __forceinline__ void store_rows(const G9_LDS unsigned char *lds, int n, F row) {
    constexpr int V = 16 / sizeof(O), PER = COLS / V;
    typedef O OV __attribute__((ext_vector_type(V)));
    typedef O OU __attribute__((ext_vector_type(V), aligned(sizeof(O))));
    const int col = (int)threadIdx.x % PER * V;
#pragma unroll
    for (int i0 = 0; i0 < ROWS; i0 += NTH / PER) {
        const int i = i0 + (int)threadIdx.x / PER;
        O *c = row(i);
        if (!c || col >= n) continue;
        const OV v = *reinterpret_cast<const G9_LDS OV *>(lds + i * PITCH + col * sizeof(O));
        if (col + V <= n) *reinterpret_cast<OU *>(c + col) = v;
        else
#pragma unroll
            for (int j = 0; j < V; j++)
                if (col + j < n) c[col + j] = v[j];
    }
}

__device__ __forceinline__ float silu(float z) { return z / (1.f + expf(-z)); }

}  // namespace g9llm
