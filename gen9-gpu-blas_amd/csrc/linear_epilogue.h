// What a linear layer does with a product's sums before they are stored: Z = sum + bias, Y = R + dropout(act(Z)), all in FP32,
// Y and Z each rounded once.
//
// Three kinds of activation, chosen once outside the loops over a tile: z < low ? low : z (none: low = −∞, ReLU: 0);
// z·σ(a·z + b·z³) (SiLU: a = 1, b = 0; GELU's tanh form, 0.5·z·(1 + tanh(c·(z + 0.044715·z³))) with c = √(2/π): a = 2c, b =
// 2c·0.044715, as 0.5·(1 + tanh x) = σ(2x)); and z·Φ(z), GELU itself.
#pragma once
#include "dropout.h"
#include "rows.h"
#include <type_traits>

namespace g9llm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
enum Kind { KIND_CLIP, KIND_SIGMOID, KIND_ERF };

struct Activation {
    int kind;
    float low, a, b;
};
inline Activation make_act(int act) {
    switch (act) {
    case GEN9BLAS_ACT_RELU: return {KIND_CLIP, 0.f, 0.f, 0.f};
    case GEN9BLAS_ACT_GELU: return {KIND_ERF, 0.f, 0.f, 0.f};
    case GEN9BLAS_ACT_GELU_TANH: return {KIND_SIGMOID, 0.f, 1.5957691216057308f, 0.0713548162726009f};
    case GEN9BLAS_ACT_SILU: return {KIND_SIGMOID, 0.f, 1.f, 0.f};
    }
    return {KIND_CLIP, -INFINITY, 0.f, 0.f};
}

// T: the type of the result. For FP16 the hardware's exponential and reciprocal are enough: a step of 2^-23 of the value each, and the
// rounding of the exponential's argument adds |x| units of 2^-24 where x < 0 (2^-20 at −16, where z·sigmoid is a subnormal FP16 number).
template <class T> __device__ __forceinline__ float sigmoid(float x) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
    else return 1.f / (1.f + expf(-x));
}
// The normal distribution function, and its density. For FP16: with t = |z|, Φ(−t) = e^(−t²/2)·h(t), h(t) = erfcx(t/√2)/2 a
// polynomial without constant term in 1 / (1 + 0.26 t), fitted here to 2^-25 of h over t = 0..14 (least squares, reweighted by the
// error); the exponential's argument adds t² units of 2^-24. erfcf and expf take 102 of the 2048 × 11008 gradient's µs, this 31.
template <class T> __device__ __forceinline__ float phi(float z, float *density = nullptr) {
    if constexpr (sizeof(T) == 2) {
        const float e = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z), u = __builtin_amdgcn_rcpf(__builtin_fmaf(0.26f, fabsf(z), 1.f));
        float h = 0.030504918017258263f;
        h = __builtin_fmaf(h, u, -0.15282897932830952f);
        h = __builtin_fmaf(h, u, 0.25149159502565716f);
        h = __builtin_fmaf(h, u, -0.15094929368823687f);
        h = __builtin_fmaf(h, u, 0.16094806642182638f);
        h = __builtin_fmaf(h, u, 0.05102760111770026f);
        h = __builtin_fmaf(h, u, 0.10303027175292723f);
        h = __builtin_fmaf(h, u, 0.1030167483806316f);
        h = __builtin_fmaf(h, u, 0.10375905992855701f);
        const float q = h * u * e;
        if (density) *density = 0.3989422804014327f * e;
        return z < 0.f ? q : 1.f - q;
    } else {
        if (density) *density = 0.3989422804014327f * expf(-0.5f * z * z);
        return 0.5f * erfcf(-0.7071067811865476f * z);
    }
}

// z² with an end, so that its product with b = 0, or with the zero of a slope far out, is none of infinity's.
__device__ __forceinline__ float square(float z) { return fminf(z * z, 1e30f); }

template <class T, int KIND> __device__ __forceinline__ float activate(const Activation &act, float z) {
    if constexpr (KIND == KIND_CLIP) return z < act.low ? act.low : z;
    if constexpr (KIND == KIND_SIGMOID) return z * sigmoid<T>(z * (act.a + act.b * square(z)));
    return z * phi<T>(z);
}
// dy times d activate / dz; what ReLU clips is zero, whatever dy is. An infinite z, as FP16's stored ones past 65504 are, has the slope
// that they have, 0 or 1: a factor that is zero there takes a z with an end (a NaN stays in s and p).
template <class T, int KIND> __device__ __forceinline__ float gradient(const Activation &act, float dy, float z) {
    if constexpr (KIND == KIND_CLIP) return z > act.low || z != z ? dy : 0.f;
    if constexpr (KIND == KIND_SIGMOID) {
        const float q = square(z), s = sigmoid<T>(z * (act.a + act.b * q));
        return dy * (s + __builtin_amdgcn_fmed3f(z, -3e38f, 3e38f) * s * (1.f - s) * (act.a + 3.f * act.b * q));
    }
    float density;
    const float p = phi<T>(z, &density);
    return dy * __builtin_fmaf(__builtin_amdgcn_fmed3f(z, -3e38f, 3e38f), density, p);
}

template <class T> struct Epilogue {
    const float *bias;   // or null
    T *Z;                // or null
    const T *R;          // or null
    long long ldz, ldr;
    Activation act;
    Dropout dropout;
    int past = 0;        // results go out past the caches

    template <int V> struct Cols { float bias[V]; };
    template <int V> struct Res {
        typedef T Vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
        Vec v;
    };

    // Keeps the loads of these kernel arguments before this place.
    __device__ __forceinline__ void pin() {
        asm volatile("" : "+s"(bias), "+s"(Z), "+s"(R), "+s"(ldz), "+s"(ldr), "+s"(act.kind), "+s"(act.low), "+s"(act.a), "+s"(act.b));
        asm volatile("" : "+s"(dropout.limit), "+s"(dropout.scale), "+s"(dropout.seed[0]), "+s"(dropout.seed[1]), "+s"(dropout.offset[0]), "+s"(dropout.offset[1]), "+s"(past));
    }
    template <class F> __device__ __forceinline__ void each(F f) const {
        if (act.kind == KIND_CLIP) f(std::integral_constant<int, KIND_CLIP>{});
        else if (act.kind == KIND_SIGMOID) f(std::integral_constant<int, KIND_SIGMOID>{});
        else f(std::integral_constant<int, KIND_ERF>{});
    }
    // Columns n .. n + V − 1, of which `valid` exist (also none: nothing is read then).
    template <int V> __device__ __forceinline__ Cols<V> columns(int n, int valid) const {
        Cols<V> c;
        if (bias) load_some<V>(bias + n, valid, c.bias);
        else
#pragma unroll
            for (int e = 0; e < V; e++) c.bias[e] = 0.f;
        return c;
    }
    // The residual's, which a kernel asks for some rows before their sums are due (there may be none: m >= M, or valid <= 0).
    template <int V> __device__ __forceinline__ Res<V> residual(int m, int M, int n, int valid) const {
        Res<V> r = {};
        if (!R || m >= M) return r;
        const T *p = R + m * ldr + n;
        if (valid >= V) r.v = *reinterpret_cast<const typename Res<V>::Vec *>(p);
        else
#pragma unroll
            for (int e = 0; e < V; e++)
                if (e < valid) r.v[e] = p[e];
        return r;
    }
    // Row m, columns n .. n + V − 1 (n a multiple of V) from their sums: four, or eight in `v` and `hi`.
    template <class O, int V, class K> __device__ __forceinline__ void row(K, O *Y, long long ldy, int m, int n, const Cols<V> &cols, const Res<V> &res, int valid, f32x4 v, f32x4 hi = {}) const {
        if (valid <= 0) return;
        float x[V];
#pragma unroll
        for (int e = 0; e < V; e++) x[e] = (e < 4 ? v[e & 3] : hi[e & 3]) + cols.bias[e];
        auto store = [&](T *p) {
            if (past) store_some<V, T, true>(p, valid, x);
            else store_some<V>(p, valid, x);
        };
        if (Z) store(Z + m * ldz + n);
#pragma unroll
        for (int e = 0; e < V; e++) x[e] = activate<T, K::value>(act, x[e]);
        if (dropout.limit) drop<V>(dropout, m, n, x);
        if (R)
#pragma unroll
            for (int e = 0; e < V; e++) x[e] += (float)res.v[e];
        store(Y + m * ldy + n);
    }
    // One element.
    template <class O> __device__ __forceinline__ void one(O *Y, long long ldy, int m, int n, float sum) const {
        float x = sum + (bias ? bias[n] : 0.f);
        if (Z) Z[m * ldz + n] = (T)x;
        each([&](auto kind) { x = activate<T, decltype(kind)::value>(act, x); });
        if (dropout.limit) x = kept(dropout, philox(dropout, (unsigned)n >> 3, m), n & 7) ? x * dropout.scale : 0.f;
        if (R) x += (float)R[m * ldr + n];
        Y[m * ldy + n] = (T)x;
    }
};

}  // namespace g9llm
