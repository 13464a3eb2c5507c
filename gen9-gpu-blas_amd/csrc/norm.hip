// Layer norm over the rows of a matrix (gen9blas_layer_norm) and its gradients (gen9blas_layer_norm_backward).
#include "llm.h"
#include "colsum.h"
#include "rows.h"
#include <algorithm>
#include <type_traits>

namespace g9llm {

// A row is in the registers of L threads, C pieces of 16 bytes each, so that it is read once: its mean, the squares around it (the
// second pass that a variance needs, without a second read) and its result come from there. L is 16, a wave, 256, 512 or 1024.
// HBM bounds it where there are rows enough. 8192 × 4096 FP16: forward 29 µs, 134 MB at 4.6 TB/s (a copy of 1 GiB: 5.2); backward
// 39, 201 MB at 5.2, and 4.8 for the sums of its blocks. 2047 × 2501 FP32 12, 18 and 4.
template <class T> struct Piece {
    static constexpr int V = 16 / sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    // Elements n .. n + V − 1 of a row of N, zeros past its end. TAIL: the row may end inside a piece.
    template <bool TAIL = true> static __device__ __forceinline__ Vec load(const T *row, int n, int N) {
        if (n <= N - V) return *reinterpret_cast<const Vec *>(row + n);
        Vec v = {};
        if constexpr (TAIL)
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = n + e < N ? row[n + e] : T(0);
        return v;
    }
};
// How many of V elements are left to a loop that has some left.
template <bool TAIL, int V> __device__ __forceinline__ int some(int valid) { return TAIL ? valid : V; }
// Sums of `v` over the L threads of a row, in all of them. part: the row's L / 64 · K floats of LDS, that no other sum uses before a barrier.
template <int L, int K> __device__ __forceinline__ void row_sum(float *v, float *part) {
#pragma unroll
    for (int d = 1; d < (L < 64 ? L : 64); d <<= 1)
#pragma unroll
        for (int k = 0; k < K; k++) v[k] += __shfl_xor(v[k], d);
    if constexpr (L > 64) {
        const int w = (threadIdx.x >> 6) % (L / 64);
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) part[w * K + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            v[k] = 0.f;
#pragma unroll 8   // all of 16 waves' at once cost 1024 threads 40 registers each
            for (int i = 0; i < L / 64; i++) v[k] += part[i * K + k];
        }
    }
}

// y = (x − mean)·rstd·gamma + beta, rstd = 1 / √(mean((x − mean)²) + eps). The mean of x − mean, what rounding has left of it, is
// taken off again: a row whose mean is large against its values loses nothing that x has.
template <class T, int L, int C, bool TAIL>
__global__ void __launch_bounds__(L > 256 ? L : 256) norm_kernel(const T *__restrict__ X, long long ldx, const float *__restrict__ gamma, const float *__restrict__ beta, float eps,
                                                                 int M, int N, T *__restrict__ Y, long long ldy, float *__restrict__ stats) {
    using P = Piece<T>;
    constexpr int V = P::V, ROWS = (L > 256 ? L : 256) / L;
    constexpr bool KEEP = C * V <= 16;   // gamma and beta stay in registers from row to row
    __shared__ float part[2][L > 64 ? 3 * (L / 64) : 1];
    const int t = threadIdx.x % L;
    const float inv = 1.f / N;
    float g[KEEP ? C : 1][V], b[KEEP ? C : 1][V];
    auto weights = [&](int c, float *gc, float *bc) {
        const int n = (c * L + t) * V, valid = some<TAIL, V>(N - n);
#pragma unroll
        for (int e = 0; e < V; e++) gc[e] = 1.f, bc[e] = 0.f;
        if (n >= N) return;
        if (gamma) load_some<V>(gamma + n, valid, gc);
        if (beta) load_some<V>(beta + n, valid, bc);
    };
    if constexpr (KEEP)
#pragma unroll
        for (int c = 0; c < C; c++) weights(c, g[c], b[c]);
    int flip = 0;
    for (long long m0 = (long long)blockIdx.x * ROWS; m0 < M; m0 += (long long)gridDim.x * ROWS, flip ^= 1) {
        const long long m = m0 + threadIdx.x / L;
        if (L <= 64 && m >= M) break;   // whole rows of threads, and no barrier below
        const T *x = X + m * ldx;
        typename P::Vec v[C];
#pragma unroll
        for (int c = 0; c < C; c++) v[c] = P::template load<TAIL>(x, (c * L + t) * V, N);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < V; e++) s[0] += (float)v[c][e];
        row_sum<L, 1>(s, part[flip]);
        const float mean = s[0] * inv;
        s[0] = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int valid = N - (c * L + t) * V;
            if (valid <= 0) break;
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float d = !TAIL || e < valid ? (float)v[c][e] - mean : 0.f;
                s[0] += d, s[1] = __builtin_fmaf(d, d, s[1]);
            }
        }
        row_sum<L, 2>(s, part[flip] + (L > 64 ? L / 64 : 0));
        const float left = s[0] * inv, rstd = 1.f / sqrtf(fmaxf(s[1] * inv - left * left, 0.f) + eps);
        if (stats && t == 0) *reinterpret_cast<float2 *>(stats + 2 * m) = float2{mean + left, rstd};
        T *y = Y + m * ldy;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int n = (c * L + t) * V, valid = some<TAIL, V>(N - n);
            if (n >= N) break;
            float gn[V], bn[V];
            if constexpr (!KEEP) weights(c, gn, bn);
#pragma unroll
            for (int e = 0; e < V; e++) bn[e] = __builtin_fmaf((((float)v[c][e] - mean) - left) * rstd, KEEP ? g[KEEP ? c : 0][e] : gn[e], KEEP ? b[KEEP ? c : 0][e] : bn[e]);
            store_some<V>(y + n, valid, bn);
        }
    }
}
// Rows too long for the registers of a workgroup: three passes over memory.
template <class T>
__global__ void __launch_bounds__(1024) norm_long_kernel(const T *__restrict__ X, long long ldx, const float *__restrict__ gamma, const float *__restrict__ beta, float eps, int N,
                                                         T *__restrict__ Y, long long ldy, float *__restrict__ stats) {
    using P = Piece<T>;
    constexpr int V = P::V;
    __shared__ float part[48];
    const T *x = X + (long long)blockIdx.x * ldx;
    T *y = Y + (long long)blockIdx.x * ldy;
    float s[2] = {0.f, 0.f};
    for (long long n = threadIdx.x * V; n < N; n += 1024 * V) {
        const typename P::Vec v = P::load(x, (int)n, N);
#pragma unroll
        for (int e = 0; e < V; e++) s[0] += (float)v[e];
    }
    row_sum<1024, 1>(s, part);
    const float inv = 1.f / N, mean = s[0] * inv;
    s[0] = 0.f;
    for (long long n = threadIdx.x * V; n < N; n += 1024 * V) {
        const typename P::Vec v = P::load(x, (int)n, N);
#pragma unroll
        for (int e = 0; e < V; e++) {
            const float d = n + e < N ? (float)v[e] - mean : 0.f;
            s[0] += d, s[1] = __builtin_fmaf(d, d, s[1]);
        }
    }
    row_sum<1024, 2>(s, part + 16);
    const float left = s[0] * inv, rstd = 1.f / sqrtf(fmaxf(s[1] * inv - left * left, 0.f) + eps);
    if (stats && threadIdx.x == 0) *reinterpret_cast<float2 *>(stats + 2LL * blockIdx.x) = float2{mean + left, rstd};
    for (long long n = threadIdx.x * V; n < N; n += 1024 * V) {
        const typename P::Vec v = P::load(x, (int)n, N);
        const int valid = (int)(N - n);
        float g[V], b[V];
        if (gamma) load_some<V>(gamma + n, valid, g);
        if (beta) load_some<V>(beta + n, valid, b);
#pragma unroll
        for (int e = 0; e < V; e++) {
            const float z = (((float)v[e] - mean) - left) * rstd;
            b[e] = (gamma ? z * g[e] : z) + (beta ? b[e] : 0.f);
        }
        store_some<V>(y + n, valid, b);
    }
}

struct BackArgs {
    const void *dY, *X;
    long long lddy, ldx;
    const float *stats, *gamma;
    int M, N;
    void *dX;              // or null
    long long lddx;
    float *sums;           // or null: rows of 2N, the sums of dy·x̂ and of dy of each workgroup's rows
    float *dgamma, *dbeta; // where one workgroup has all rows: the results (each may be null), and no sums
    int accumulate;
};
// What the rounding of a row's mean to one FP32 number has left in z = (x − mean)·rstd, from the sum of z: at most a step of the mean.
// More than that is not the mean's, but z's own roundings, which lie on one side where x has fewer bits than the mean.
__device__ __forceinline__ float mean_left(float z, float inv, float mean, float rstd) {
    const float most = fabsf(mean) * rstd * 0x1p-23f;
    return fminf(fmaxf(z * inv, -most), most);
}
// dx = rstd·(g − mean(g) − x̂·mean(g·x̂)), g = dy·gamma, x̂ = (x − mean)·rstd, and the sums over the rows that dgamma and dbeta
// need, from one read of x and dy. stats hold the mean as one FP32 number, whose rounding is all of x̂'s error in a row far from zero
// (mean 2^18 times the spread: 2^-7); so what it leaves is added up with the others, and taken off: x̂ = z − off, z = (x − mean)·rstd,
// off = mean(z), mean(g·x̂) = mean(g·z) − off·mean(g). The workgroups go through the rows with a stride; a thread adds up its own
// columns, and the row groups of a workgroup are added in their order.
template <class T, int L, int C, int B, bool TAIL>
__global__ void __launch_bounds__(B) norm_back_kernel(BackArgs a) {
    using P = Piece<T>;
    constexpr int V = P::V, ROWS = B / L;
    constexpr bool KEEP = C * V <= 16;   // gamma stays in registers from row to row
    __shared__ float part[2][L > 64 ? 3 * (B / 64) : 1];
    __shared__ float join[ROWS > 1 ? 2 * V : 1][ROWS > 2 ? B + 64 / V : ROWS > 1 ? L : 1];   // reads of V by 64 / V lie in different banks
    const int t = threadIdx.x % L, group = threadIdx.x / L, N = a.N;
    const float inv = 1.f / N;
    float sg[C][V] = {}, sb[C][V] = {};
    int flip = 0;
    float keep[KEEP ? C : 1][V];
    auto weights = [&](int c, float *g) {
        const int n = (c * L + t) * V;
#pragma unroll
        for (int e = 0; e < V; e++) g[e] = 1.f;
        if (a.gamma && n < N) load_some<V>(a.gamma + n, some<TAIL, V>(N - n), g);
    };
    if constexpr (KEEP)
#pragma unroll
        for (int c = 0; c < C; c++) weights(c, keep[c]);
    for (long long m0 = (long long)blockIdx.x * ROWS; m0 < a.M; m0 += (long long)gridDim.x * ROWS, flip ^= 1) {
        const bool is = ROWS == 1 || m0 + group < a.M;   // a row group without a row goes along where the others wait for it
        if (L <= 64 && !is) break;
        const long long m = is ? m0 + group : a.M - 1;
        const T *x = (const T *)a.X + m * a.ldx, *dy = (const T *)a.dY + m * a.lddy;
        const float2 st = *reinterpret_cast<const float2 *>(a.stats + 2 * m);
        const float mean = st.x, rstd = st.y;
        typename P::Vec vx[C], vd[C];
#pragma unroll
        for (int c = 0; c < C; c++) vx[c] = P::template load<TAIL>(x, (c * L + t) * V, N), vd[c] = P::template load<TAIL>(dy, (c * L + t) * V, N);
        float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int n = (c * L + t) * V;
            if (n >= N || (L > 64 && !is)) break;
            float g[V];
            if constexpr (!KEEP) weights(c, g);
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float d = (float)vd[c][e], z = ((float)vx[c][e] - mean) * rstd, w = d * (KEEP ? keep[KEEP ? c : 0][e] : g[e]);
                sb[c][e] += d, s[0] += w, s[1] = __builtin_fmaf(w, z, s[1]), s[2] += !TAIL || n + e < N ? z : 0.f;
            }
        }
        if (!a.dX && !a.dgamma) continue;
        row_sum<L, 3>(s, part[flip] + (L > 64 ? group * (L / 64) * 3 : 0));
        // z and dy's FP32 values are made again from here: kept over the sum they cost FP16 rows 24 registers of each thread's 128, and spills
#pragma unroll
        for (int c = 0; c < C; c++) asm volatile("" : "+v"(vx[c]), "+v"(vd[c]));
        const float off = mean_left(s[2], inv, mean, rstd), p = s[0] * inv, q = (s[1] - off * s[0]) * inv;
        T *dx = (T *)a.dX + m * a.lddx;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int n = (c * L + t) * V, valid = some<TAIL, V>(N - n);
            if (n >= N || (L > 64 && !is)) break;
            float g[V];
            if constexpr (!KEEP) weights(c, g);
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float d = (float)vd[c][e], xh = __builtin_fmaf((float)vx[c][e] - mean, rstd, -off);
                g[e] = rstd * (d * (KEEP ? keep[KEEP ? c : 0][e] : g[e]) - p - xh * q);
                sg[c][e] = __builtin_fmaf(d, xh, sg[c][e]);
            }
            if (a.dX) store_some<V>(dx + n, valid, g);
        }
    }
    if (!a.sums && !a.dgamma && !a.dbeta) return;
    if constexpr (ROWS > 2) {
#pragma unroll
        for (int c = 0; c < C; c++) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; e++) join[e][threadIdx.x] = sg[c][e], join[V + e][threadIdx.x] = sb[c][e];
            __syncthreads();
            for (int o = threadIdx.x; o < 2 * V * L; o += B) {
                const int beta = o / (V * L), at = o % (V * L), n = c * V * L + at;
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < ROWS; r++) sum += join[beta * V + at % V][r * L + at / V];
                if (n >= N) continue;
                float *out = a.sums ? a.sums + (2LL * blockIdx.x + beta) * N : beta ? a.dbeta : a.dgamma;
                if (out) out[n] = !a.sums && a.accumulate ? out[n] + sum : sum;
            }
        }
        return;
    }
    if constexpr (ROWS == 2) {
#pragma unroll
        for (int c = 0; c < C; c++) {
            __syncthreads();
            if (group)
#pragma unroll
                for (int e = 0; e < V; e++) join[e][t] = sg[c][e], join[V + e][t] = sb[c][e];
            __syncthreads();
            if (!group)
#pragma unroll
                for (int e = 0; e < V; e++) sg[c][e] += join[e][t], sb[c][e] += join[V + e][t];
        }
        if (group) return;
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int n = (c * L + t) * V, valid = some<TAIL, V>(N - n);
        if (n >= N) break;
        auto put = [&](float *out, float *v) {
            if (!out) return;
            float old[V];
            if (!a.sums && a.accumulate) {
                load_some<V>(out + n, valid, old);
#pragma unroll
                for (int e = 0; e < V; e++) v[e] += old[e];
            }
            store_some<V>(out + n, valid, v);
        };
        put(a.sums ? a.sums + 2LL * blockIdx.x * N : a.dgamma, sg[c]);
        put(a.sums ? a.sums + (2LL * blockIdx.x + 1) * N : a.dbeta, sb[c]);
    }
}

// Rows too long for that: dx and off of each row (each may be null), from two passes over x and dy, and the sums by themselves.
template <class T>
__global__ void __launch_bounds__(1024) norm_back_long_kernel(BackArgs a, float *__restrict__ offs) {
    using P = Piece<T>;
    constexpr int V = P::V;
    __shared__ float part[48];
    const T *x = (const T *)a.X + blockIdx.x * a.ldx, *dy = (const T *)a.dY + blockIdx.x * a.lddy;
    T *dx = (T *)a.dX + blockIdx.x * a.lddx;
    const float mean = a.stats[2LL * blockIdx.x], rstd = a.stats[2LL * blockIdx.x + 1], inv = 1.f / a.N;
    float s[3] = {0.f, 0.f, 0.f};
    auto each = [&](auto use) {
        for (long long n = threadIdx.x * V; n < a.N; n += 1024 * V) {
            const typename P::Vec vx = P::load(x, (int)n, a.N), vd = P::load(dy, (int)n, a.N);
            const int valid = (int)(a.N - n);
            float g[V], z[V];
            if (a.gamma) load_some<V>(a.gamma + n, valid, g);
#pragma unroll
            for (int e = 0; e < V; e++) g[e] = a.gamma ? (float)vd[e] * g[e] : (float)vd[e], z[e] = ((float)vx[e] - mean) * rstd;
            use(n, valid, g, z);
        }
    };
    each([&](long long, int valid, const float *g, const float *z) {
#pragma unroll
        for (int e = 0; e < V; e++) s[0] += g[e], s[1] += e < valid ? g[e] * z[e] : 0.f, s[2] += e < valid ? z[e] : 0.f;
    });
    row_sum<1024, 3>(s, part);
    const float off = mean_left(s[2], inv, mean, rstd), p = s[0] * inv, q = (s[1] - off * s[0]) * inv;
    if (offs && threadIdx.x == 0) offs[blockIdx.x] = off;
    if (!a.dX) return;
    each([&](long long n, int valid, float *g, const float *z) {
#pragma unroll
        for (int e = 0; e < V; e++) g[e] = rstd * (g[e] - p - (z[e] - off) * q);
        store_some<V>(dx + n, valid, g);
    });
}
// offs: null where dbeta alone is wanted
template <class T>
__global__ void __launch_bounds__(256) norm_sums_long_kernel(BackArgs a, const float *__restrict__ offs, int rows) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= a.N) return;
    const long long m0 = (long long)blockIdx.y * rows, m1 = min(m0 + rows, (long long)a.M);
    float g = 0.f, b = 0.f;
    const T *dy = (const T *)a.dY + n, *x = (const T *)a.X + n;
    if (offs)
        for (long long m = m0; m < m1; m++) {
            const float d = (float)dy[m * a.lddy];
            g = __builtin_fmaf(d, ((float)x[m * a.ldx] - a.stats[2 * m]) * a.stats[2 * m + 1] - offs[m], g), b += d;
        }
    else
        for (long long m = m0; m < m1; m++) b += (float)dy[m * a.lddy];
    a.sums[2LL * blockIdx.y * a.N + n] = g;
    a.sums[(2LL * blockIdx.y + 1) * a.N + n] = b;
}

// f(L, C, TAIL) for rows of N elements of T by the first pair of threads and pieces that holds them, or false.
template <int L_, int C_> struct Shape { static constexpr int L = L_, C = C_; };
template <class T, class F, class... S> static bool by_length(int N, F f, S... shapes) {
    constexpr int V = 16 / (int)sizeof(T);
    auto take = [&](auto s) {
        if (cdiv(N, V) > s.L * s.C) return false;
        if (N % V) f(s, std::true_type{});
        else f(s, std::false_type{});
        return true;
    };
    return (take(shapes) || ...);
}

template <class T>
static int norm(int M, int N, const T *X, int ldx, const float *gamma, const float *beta, float eps, T *Y, int ldy, float *stats) {
    int rc = 0;
    const bool fits = by_length<T>(N, [&](auto shape, auto tail) {
        constexpr int L = shape.L, C = shape.C, B = L > 256 ? L : 256, ROWS = B / L;
        const long long blocks = std::min(cdiv(M, ROWS), 1536LL / B * num_cus);   // as many as run at once
        hipLaunchKernelGGL((norm_kernel<T, L, C, tail()>), dim3((unsigned)blocks), dim3(B), 0, stream, X, ldx, gamma, beta, eps, M, N, Y, ldy, stats);
        const hipError_t e = hipGetLastError();
        rc = e == hipSuccess ? 0 : hip_fail(e, "norm_kernel", __FILE__, __LINE__);
    }, Shape<16, 1>(), Shape<16, 2>(), Shape<64, 1>(), Shape<64, 2>(), Shape<64, 4>(), Shape<256, 2>(), Shape<256, 4>(), Shape<256, 8>(), Shape<1024, 4>());
    if (fits) return rc;
    return by_rows(M, 1024, [&](long long m0, unsigned rows) -> int {
        hipLaunchKernelGGL((norm_long_kernel<T>), dim3(rows), dim3(1024), 0, stream, X + m0 * ldx, ldx, gamma, beta, eps, N, Y + m0 * ldy, ldy, stats ? stats + 2 * m0 : nullptr);
        G9_HIP(hipGetLastError());
        return 0;
    });
}
template <class T> static int norm_back(BackArgs a) {
    int rc = 0;
    void *sums = nullptr;
    float *dgamma = a.dgamma, *dbeta = a.dbeta;
    const bool both = dgamma || dbeta;
    const bool fits = by_length<T>(a.N, [&](auto shape, auto tail) {
        constexpr int L = shape.L, C = shape.C, B = L > 512 ? L : 512, ROWS = B / L;
        const int blocks = (int)std::min(cdiv(a.M, 4LL * ROWS), (long long)num_cus * (1024 / B));
        auto run = [&]() -> int {
            if (both && blocks > 1) {
                G9_TRY(work_buffer("layer_norm_backward", SLOT_SUMS, (size_t)blocks * 2 * a.N * 4, &sums));
                a.sums = (float *)sums;
            }
            hipLaunchKernelGGL((norm_back_kernel<T, L, C, B, tail()>), dim3(blocks), dim3(B), 0, stream, a);
            G9_HIP(hipGetLastError());
            return a.sums ? column_sums((float *)sums, blocks, a.N, 2LL * a.N, dgamma, dbeta, a.accumulate) : 0;
        };
        rc = run();
    }, Shape<16, 1>(), Shape<16, 2>(), Shape<64, 1>(), Shape<64, 2>(), Shape<256, 1>(), Shape<256, 2>(), Shape<512, 2>(), Shape<1024, 2>());
    if (fits) return rc;
    const int rows = (int)std::max(32LL, cdiv(a.M, 512));
    const long long blocks = cdiv(a.M, rows);
    float *offs = nullptr;
    if (both) {   // before the first launch: what is refused has written nothing
        const long long planes = blocks * 2 * a.N;
        G9_TRY(work_buffer("layer_norm_backward", SLOT_SUMS, (size_t)(planes + a.M) * 4, &sums));
        a.sums = (float *)sums;
        if (dgamma) offs = a.sums + planes;
    }
    if (a.dX || offs)
        G9_TRY(by_rows(a.M, 1024, [&](long long m0, unsigned rows) -> int {
            BackArgs b = a;
            b.dY = (const T *)a.dY + m0 * a.lddy, b.X = (const T *)a.X + m0 * a.ldx, b.stats = a.stats + 2 * m0;
            if (a.dX) b.dX = (T *)a.dX + m0 * a.lddx;
            hipLaunchKernelGGL((norm_back_long_kernel<T>), dim3(rows), dim3(1024), 0, stream, b, offs ? offs + m0 : nullptr);
            G9_HIP(hipGetLastError());
            return 0;
        }));
    if (both) {
        hipLaunchKernelGGL((norm_sums_long_kernel<T>), dim3((unsigned)cdiv(a.N, 256), (unsigned)blocks), dim3(256), 0, stream, a, (const float *)offs, rows);
        G9_HIP(hipGetLastError());
        G9_TRY(column_sums((float *)sums, blocks, a.N, 2LL * a.N, dgamma, dbeta, a.accumulate));
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
    const BackArgs a = {dY, X, lddy, ldx, stats, gamma, M, N, dX, lddx, nullptr, dgamma, dbeta, accumulate};
    return type == GEN9BLAS_H ? norm_back<_Float16>(a) : norm_back<float>(a);
}

}  // extern "C"
