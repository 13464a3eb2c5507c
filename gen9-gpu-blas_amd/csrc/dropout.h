// Dropout from a counter-based generator: which elements a matrix loses is a function of their place, a seed and an offset,
// so that the mask is never stored and the backward pass computes it again.
//
// The generator is Philox4x32 of ten rounds (Salmon, Moraes, Dror, Shaw: Parallel Random Numbers: As Easy as 1, 2, 3, 2011): a
// round multiplies two of the four words by constants to 64 bits and mixes the halves with the others and the key. The
// counter of columns 8c .. 8c+7 of row r is (c, r, offset, offset >> 32), the key (seed, seed >> 32), and the eight columns
// take the 16-bit parts of its four words, low ones first. An element is lost if its part is below limit = round(65536 p),
// the others are scaled by 65536 / (65536 − limit): the share is p to the nearest of 2^-16, and the scale is that share's.
// 16 bits an element: ten rounds for each 8 elements are as many instructions as memory leaves time for at 2 bytes read and 2
// written; of 32 bits they would be twice that.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace g9llm {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct Dropout {
    unsigned limit;   // 0: none
    float scale;
    unsigned seed[2], offset[2];
};
// p in [0, 1]
inline Dropout make_dropout(double p, uint64_t seed, uint64_t offset) {
    const unsigned limit = (unsigned)nearbyint(p * 65536);
    return {limit, limit < 65536 ? (float)(65536.0 / (65536 - limit)) : 0.f, {(unsigned)seed, (unsigned)(seed >> 32)}, {(unsigned)offset, (unsigned)(offset >> 32)}};
}

__device__ __forceinline__ u32x4 philox(const Dropout &d, unsigned group, unsigned row) {
    unsigned c0 = group, c1 = row, c2 = d.offset[0], c3 = d.offset[1], k0 = d.seed[0], k1 = d.seed[1];
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c1 = (unsigned)b, c3 = (unsigned)a;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}
// Whether the element of the group's column e (0..7) stays.
__device__ __forceinline__ bool kept(const Dropout &d, u32x4 words, int e) { return (words[e >> 1] >> 16 * (e & 1) & 0xffffu) >= d.limit; }
// v[0 .. V-1] are columns n .. n + V − 1 of a row (n a multiple of V, V 4 or 8): lost ones become zeros, whatever they were.
template <int V> __device__ __forceinline__ void drop(const Dropout &d, unsigned row, int n, float *v) {
    const u32x4 w = philox(d, (unsigned)n >> 3, row);
    const u32x4 mine = V == 4 && (n & 4) ? u32x4{w[2], w[3], 0, 0} : w;
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = kept(d, mine, e) ? v[e] * d.scale : 0.f;
}

}  // namespace g9llm
