// Launches over the rows of long matrices, and vectors of rows at element alignment.
#pragma once
#include "llm.h"
#include <algorithm>

namespace g9llm {

// f(first row, rows) for all M rows, in launches whose threads a launch can index at a workgroup of `threads` a row.
template <class F> static int by_rows(long long M, int threads, F f) {
    const long long most = 0xffffffffLL / threads;
    for (long long m0 = 0; m0 < M; m0 += most) G9_TRY(f(m0, (unsigned)std::min(M - m0, most)));
    return 0;
}

// V consecutive elements at element alignment, of which `valid` exist; zeros for the others.
template <int V, class T> __device__ __forceinline__ void load_some(const T *p, int valid, float *v) {
    typedef T TV __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    if (valid >= V) {
        const TV q = *reinterpret_cast<const TV *>(p);
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = (float)q[e];
    } else
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = e < valid ? (float)p[e] : 0.f;
}
// PAST: past the caches, for what nothing reads soon.
template <int V, class T, bool PAST = false> __device__ __forceinline__ void store_some(T *p, int valid, const float *v) {
    typedef T TV __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    if (valid >= V) {
        TV q;
#pragma unroll
        for (int e = 0; e < V; e++) q[e] = (T)v[e];
        if constexpr (PAST) __builtin_nontemporal_store(q, reinterpret_cast<TV *>(p));
        else *reinterpret_cast<TV *>(p) = q;
    } else
#pragma unroll
        for (int e = 0; e < V; e++)
            if (e < valid) p[e] = (T)v[e];
}

}  // namespace g9llm
