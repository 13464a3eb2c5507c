// Mixture of experts: the router (gen9blas_moe_route) and the products of each token's experts (gen9blas_moe_gemm).
#include "mx4_tile_kernel.h"
#include "mx4_rows_kernel.h"
#include <algorithm>

namespace g9llm {

constexpr int MAX_EXPERTS = 1024, MAX_K = 64;

struct RouteArgs {
    const void *logits;
    long long ldl;
    const float *bias;
    int T, E, sigmoid, groups, top_groups, k, renorm;
    float scale;
    int *ids;
    float *weights;
};

// An order on floats (no NaN) as unsigned numbers; −0 and +0 are equal after adding +0.
__device__ __forceinline__ unsigned ordered(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Reductions over the 64 lanes by DPP: within rows of 16, then from each row to the next; lane 63 has the result, which all get.
// (Six exchanges through LDS permutes, for each of k choices, were most of 8192 tokens' 21 µs.)
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned dpp(unsigned old, unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, ROWS, 0xf, false);
}
template <class F> __device__ __forceinline__ unsigned wave_reduce(unsigned v, unsigned identity, F op) {
    v = op(v, dpp<0x111, 0xf>(identity, v));   // row_shr 1, 2, 4, 8
    v = op(v, dpp<0x112, 0xf>(identity, v));
    v = op(v, dpp<0x114, 0xf>(identity, v));
    v = op(v, dpp<0x118, 0xf>(identity, v));
    v = op(v, dpp<0x142, 0xa>(identity, v));   // lane 15 of rows 0 and 2 to rows 1 and 3
    v = op(v, dpp<0x143, 0xc>(identity, v));   // lane 31 to rows 2 and 3
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ unsigned as_u(float v) { return __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ float as_f(unsigned v) { return __builtin_bit_cast(float, v); }
__device__ __forceinline__ float wave_max(float v) {
    return as_f(wave_reduce(as_u(v), as_u(-__builtin_inff()), [](unsigned a, unsigned b) { return as_u(fmaxf(as_f(a), as_f(b))); }));
}
__device__ __forceinline__ float wave_sum(float v) {
    return as_f(wave_reduce(as_u(v), 0u, [](unsigned a, unsigned b) { return as_u(as_f(a) + as_f(b)); }));
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
    return wave_reduce(v, 0u, [](unsigned a, unsigned b) { return a > b ? a : b; });
}

// A wave routes a token: lane l holds the NL experts from l·NL on, so that of equal choices the lowest lane's, and there the
// first, is the lowest index. A lane sorts its choices (as ordered numbers; 0: not to be chosen) once, neighbours only, which keeps
// equal ones in their order; the k experts are k rounds of the wave's maximum over the lanes' first, and the lane that had it moves
// its own up. Instructions bound it: 8192 tokens of 256 experts, 8 chosen, 10.4 µs a call; 12.1 with each round over all of a lane's choices.
template <class T, int NL>
__global__ void __launch_bounds__(256) moe_route_kernel(RouteArgs a) {
    const float ninf = -__builtin_inff();
    extern __shared__ float lds[];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const long long t = (long long)blockIdx.x * 4 + wv;
    if (t >= a.T) return;   // whole waves: nothing below waits for another wave
    float *mine = lds + wv * 64 * NL;
    float score[NL], choice[NL], bias[NL];
    auto load = [&](auto *row, float *v, float none) {
        typedef std::remove_cv_t<std::remove_reference_t<decltype(*row)>> E;
        if (lane * NL + NL <= a.E) {
            E e[NL];
            __builtin_memcpy(e, row + lane * NL, sizeof e);
#pragma unroll
            for (int i = 0; i < NL; i++) v[i] = (float)e[i];
        } else
#pragma unroll
            for (int i = 0; i < NL; i++) v[i] = lane * NL + i < a.E ? (float)row[lane * NL + i] : none;
    };
    load((const T *)a.logits + t * a.ldl, score, ninf);
    if (a.bias) load(a.bias, bias, 0.f);
    bool nan = false;
#pragma unroll
    for (int i = 0; i < NL; i++) nan |= score[i] != score[i];
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const bool out = !(score[i] > ninf);
            score[i] = 1.f / (1.f + expf(-score[i]));
            choice[i] = out ? ninf : score[i];
        }
    } else {
        float m = ninf, sum = 0.f;
#pragma unroll
        for (int i = 0; i < NL; i++) m = fmaxf(m, score[i]);
        m = wave_max(m);
#pragma unroll
        for (int i = 0; i < NL; i++) {
            choice[i] = score[i] > ninf ? score[i] : ninf;
            score[i] = m > ninf ? expf(score[i] - m) : 0.f;
            sum += score[i];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int i = 0; i < NL; i++) score[i] /= sum;
        if (a.bias)
#pragma unroll
            for (int i = 0; i < NL; i++)
                if (choice[i] > ninf) choice[i] = score[i];
    }
    if (a.bias)
#pragma unroll
        for (int i = 0; i < NL; i++) {
            if (choice[i] > ninf) choice[i] += bias[i];
            if (choice[i] != choice[i]) choice[i] = ninf, nan = true;
        }
    nan = __ballot(nan) != 0;
    unsigned key[NL];
    int at[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) key[i] = choice[i] > ninf ? ordered(choice[i]) : 0, at[i] = i;
    if (a.groups > 1) {
        // `per` lanes a group (a power of two) take its choices, their own where those are the group's, and join their two largest
        const int size = a.E / a.groups;
        int per = 64;
        while (per * a.groups > 64) per >>= 1;
        const bool own = per * NL == size;
        const int group = lane / per;
        float best = ninf, second = ninf;
        auto take = [&](float b, float s) {
            second = fmaxf(fmaxf(second, s), fminf(best, b));
            best = fmaxf(best, b);
        };
        if (own) {
#pragma unroll
            for (int i = 0; i < NL; i++) take(choice[i], ninf);
        } else {
#pragma unroll
            for (int i = 0; i < NL; i++) mine[lane * NL + i] = choice[i];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // other lanes read what these wrote
            __builtin_amdgcn_wave_barrier();
            if (group < a.groups)
                for (int i = lane % per; i < size; i += per) take(mine[group * size + i], ninf);
        }
        auto join = [&](auto other) {
            const float b = as_f(other(as_u(best))), s = as_f(other(as_u(second)));
            take(b, s);
        };
        if (per > 1) join([](unsigned v) { return dpp<0xb1, 0xf>(0, v); });    // lanes 1 apart
        if (per > 2) join([](unsigned v) { return dpp<0x4e, 0xf>(0, v); });    // 2 apart
        if (per > 4) join([](unsigned v) { return dpp<0x141, 0xf>(0, v); });   // the other four of eight
        if (per > 8) join([](unsigned v) { return dpp<0x140, 0xf>(0, v); });   // the other eight of sixteen
        if (per > 16) join([](unsigned v) { return (unsigned)__shfl_xor((int)v, 16); });
        // a group with one expert left counts as that one; one with none is never chosen
        const unsigned mark = ordered(a.sigmoid && second > ninf ? best + second : best);
        int rank = 0;
        for (int j = 0; j < a.groups; j++) {
            const unsigned other = (unsigned)__builtin_amdgcn_readlane((int)mark, j * per);
            rank += other >= mark + (j >= group);   // of equal groups the first; no mark is the largest number
        }
        const unsigned long long keep = __ballot(group < a.groups && rank < a.top_groups);   // of each group `per` bits
        if (own) {
#pragma unroll
            for (int i = 0; i < NL; i++)
                if (!(keep >> lane & 1)) key[i] = 0;
        } else
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int e = lane * NL + i;
                if (e < a.E && !(keep >> (e / size * per) & 1)) key[i] = 0;
            }
        __builtin_amdgcn_wave_barrier();   // the choices in LDS have been read
    }
#pragma unroll
    for (int i = 0; i < NL; i++) mine[lane * NL + i] = score[i];
#pragma unroll
    for (int n = 0; n < NL; n++)
#pragma unroll
        for (int i = n & 1; i + 1 < NL; i += 2) {
            const bool swap = key[i + 1] > key[i];
            const unsigned high = swap ? key[i + 1] : key[i], low = swap ? key[i] : key[i + 1];
            const int first = swap ? at[i + 1] : at[i], last = swap ? at[i] : at[i + 1];
            key[i] = high, key[i + 1] = low, at[i] = first, at[i + 1] = last;
        }
    int id = -1;      // lane j: the j-th choice
    for (int j = 0; j < a.k; j++) {
        const unsigned top = wave_max(key[0]);
        if (!top) break;   // none left
        const int from = __builtin_ctzll(__ballot(key[0] == top));
        const int e = from * NL + __builtin_amdgcn_readlane(at[0], from);
        if (lane == j) id = e;
        const bool moves = lane == from;
#pragma unroll
        for (int i = 0; i < NL; i++) {
            key[i] = moves ? i + 1 < NL ? key[i + 1] : 0 : key[i];
            if (i + 1 < NL) at[i] = moves ? at[i + 1] : at[i];
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float w = id >= 0 ? mine[id] : 0.f;
    if (a.renorm) {
        const float sum = wave_sum(w);
        w = sum == 0.f ? 0.f : w / sum;
    }
    w *= a.scale;
    if (nan) w = __builtin_nanf("");
    if (lane < a.k) {
        a.ids[t * a.k + lane] = id;
        a.weights[t * a.k + lane] = w;
    }
}

// The plan of a grouped product: slots by expert (order; places whose id is no expert come last, as expert E), off[e] where
// expert e's begin, and the tiles of `rows` slots: (expert, first place), (−1, 0) past the last, their number in front. One
// workgroup: the ids are counted in LDS, a scan gives each expert's place, and the ids (the first 8192 from registers) are placed.
// Latencies bound it, so a thread has eight loads or LDS atomics on their way, none of them conditional (a rank that the count
// gives, kept in memory for the placing, took longer than counting twice: 8192 ids 14.6 µs and 8.1). The order of a group's slots
// varies from call to call; no result depends on it.
__device__ __forceinline__ int2 scan_pair(int2 v, int lane) {   // sums over the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int x = __shfl_up(v.x, d), y = __shfl_up(v.y, d);
        if (lane >= d) v.x += x, v.y += y;
    }
    return v;
}
__global__ void __launch_bounds__(1024) moe_plan_kernel(const int *__restrict__ ids, int n, int E, int rows, int *order, int *off, int *tiles, int most) {
    __shared__ int count[MAX_EXPERTS + 65], base[MAX_EXPERTS + 65];   // the last 64: lanes without an id
    __shared__ int2 waves[16];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    auto load = [&](long long i0, int *e) {
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = ids[min(i0 + j * 1024, (long long)n - 1)];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = i0 + j * 1024 < n ? (int)min((unsigned)e[j], (unsigned)E) : E + 1 + lane;
    };
    int mine8[8];
    load(t, mine8);
    for (int i = t; i <= E; i += 1024) count[i] = 0;
    __syncthreads();
    auto each = [&](auto use) {
        use((long long)t, mine8);
        for (long long i0 = 8 * 1024 + t; i0 - t < n; i0 += 8 * 1024) {
            int e[8];
            load(i0, e);
            use(i0, e);
        }
    };
    each([&](long long, const int *e) {
#pragma unroll
        for (int j = 0; j < 8; j++) atomicAdd(&count[e[j]], 1);
    });
    __syncthreads();
    const int mine = t < E ? count[t] : 0, own = (mine + rows - 1) / rows;
    const int2 s = scan_pair({mine, own}, lane);
    if (lane == 63) waves[wv] = s;
    __syncthreads();
    int2 before = {s.x - mine, s.y - own}, all = {0, 0};
#pragma unroll
    for (int w = 0; w < 16; w++) {
        const int2 v = waves[w];
        if (w < wv) before.x += v.x, before.y += v.y;
        all.x += v.x, all.y += v.y;
    }
    auto put = [&](int e, int first, int tile, int c) {
        base[e] = first, off[e] = first;
        for (int i = 0; i * rows < c; i++) tiles[2 * (tile + i)] = e, tiles[2 * (tile + i) + 1] = first + i * rows;
    };
    if (t < E) put(t, before.x, before.y, mine);
    const int last = all.y + (count[E] + rows - 1) / rows;
    if (t == 0) {
        put(E, all.x, all.y, count[E]);
        off[E + 1] = n, tiles[-1] = last;
    }
    for (int i = last + t; i < most; i += 1024) tiles[2 * i] = -1, tiles[2 * i + 1] = 0;
    __syncthreads();
    each([&](long long i0, const int *e) {
        int at[8];
#pragma unroll
        for (int j = 0; j < 8; j++) at[j] = atomicAdd(&base[e[j]], 1);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (e[j] <= E) order[at[j]] = (int)i0 + j * 1024;
    });
}

// C(t) = Σ_s weights(t, s) · y(t, s), in the order of s; places that are no expert's are left out. A thread for four columns
// of a token; y has rows of ld, whole 16-byte pieces. 2047 × 4 places, 4096 columns, FP16: 22 µs, 6.8 TB/s from HBM and the last cache.
template <class T>
__global__ void __launch_bounds__(256) moe_join_kernel(const float *__restrict__ y, long long ld, const int *__restrict__ ids, const float *__restrict__ weights,
                                                       int S, int E, int N, T *__restrict__ C, long long ldct) {
    const long long t = blockIdx.y;
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= N) return;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < S; s++) {
        const bool is = (unsigned)ids[t * S + s] < (unsigned)E;
        const float w = is ? weights[t * S + s] : 0.f;
        const f32x4 v = *reinterpret_cast<const f32x4 *>(y + (t * S + s) * ld + n);
        if (is) sum += w * v;
    }
    T *c = C + t * ldct + n;
    if (n + 4 <= N) {
        typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        *reinterpret_cast<T4 *>(c) = T4{(T)sum[0], (T)sum[1], (T)sum[2], (T)sum[3]};
    } else
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (n + j < N) c[j] = (T)sum[j];
}

template <class T> static int launch_route(const RouteArgs &a) {
    const dim3 grid((unsigned)cdiv(a.T, 4)), block(256);
    auto run = [&](auto kernel, int experts) { hipLaunchKernelGGL(kernel, grid, block, (size_t)experts * 16, stream, a); };
    if (a.E <= 64) run(moe_route_kernel<T, 1>, 64);
    else if (a.E <= 128) run(moe_route_kernel<T, 2>, 128);
    else if (a.E <= 256) run(moe_route_kernel<T, 4>, 256);
    else if (a.E <= 512) run(moe_route_kernel<T, 8>, 512);
    else run(moe_route_kernel<T, 16>, 1024);
    G9_HIP(hipGetLastError());
    return 0;
}

// The workgroups of a launch, or an error if their threads are more than it can index.
static int grid_of(long long workgroups, int threads, dim3 *grid) {
    if (workgroups * threads > 0xffffffffLL) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "moe_gemm: more tiles than one launch can index");
    *grid = dim3((unsigned)workgroups);
    return 0;
}

template <class T, class O, bool GATED> static int launch_grouped(const Rows &R, const Mx4View &W, const Mx4View &G, int E, int most, int rows, int Tn, long long n) {
    dim3 grid;
    if (rows > 32) {
        Planes A;
        const int ntiles = (int)cdiv(W.rt, GATED ? 8 : 16);
        G9_TRY(grid_of(cdiv((long long)most * ntiles, 8) * 8, 256, &grid));
        G9_TRY(stage_planes<T>(R, Tn, W.K, W.kc, &A));
        hipLaunchKernelGGL((mx4_gemm_tile_kernel<T, O, true, GATED>), grid, dim3(256), 0, stream, A, R, W, G, E, 0, ntiles);
        G9_HIP(hipGetLastError());
        return 0;
    }
    const Split whole = {1, nullptr, 0, 0};
    // few: 8 waves share the rows of a chunk, 128·NT columns a workgroup; rows: each wave has its own, 16·NT columns
    auto few = [&](auto kernel, int cols) -> int {
        const int ntiles = (int)cdiv(W.rt, cols);
        G9_TRY(grid_of(cdiv((long long)most * ntiles, 8) * 8, 512, &grid));
        hipLaunchKernelGGL(kernel, grid, dim3(512), 0, stream, R, W, G, E, most, ntiles, whole);
        G9_HIP(hipGetLastError());
        return 0;
    };
    const bool many = std::min<long long>(n, E) * cdiv(W.rt, 16) >= 2LL * num_cus;   // workgroups of 256 columns
    if constexpr (sizeof(T) == 2) {
        if (rows == 32) {
            // FP16 128 × 4 places of 64 experts, 4096 × 1536, not gated: 51.0 µs; one column tile a wave 56.4. Gated, 1536 × 4096, 87.7
            // and 77.1; 64 × 4 places of 16 experts 44.3 and 29.5
            if constexpr (!GATED) {
                if (many) return few(mx4_gemm_few_kernel<T, O, 2, 2, 4, true, GATED>, 16);
            }
            return few(mx4_gemm_few_kernel<T, O, 2, 1, 4, true, GATED>, 8);
        }
    }
    // FP32 joined, 24 × 4 places of 64 experts, 4096 × 1536: 35.6 µs; one column tile a wave 41.3, the rows kernel 63
    if (many) return few(mx4_gemm_few_kernel<T, O, 1, 2, 4, true, GATED>, 16);
    // FP16 gated, 8 places, 1536 × 4096: 13.6 µs; few kernel 20.6 and more. FP32 gated, 7 places, 864 × 3840: 14.2 µs, the few
    // kernel, whose 49 workgroups leave most CUs idle, 24
    if (std::min<long long>(n, E) * cdiv(W.rt, 8) >= num_cus) return few(mx4_gemm_few_kernel<T, O, 1, 1, 4, true, GATED>, 8);
    G9_TRY(grid_of((long long)most * W.rt, 256, &grid));
    hipLaunchKernelGGL((mx4_gemm_rows_kernel<T, O, 2, true, GATED>), grid, dim3(256), 0, stream, R, W, G, E, whole);
    G9_HIP(hipGetLastError());
    return 0;
}

template <class T>
static int join(const float *y, long long ld, const int *ids, const float *weights, int Tn, int S, int E, int N, T *C, long long ldct) {
    for (long long t0 = 0; t0 < Tn; t0 += 65535) {   // the grid's y limit
        const dim3 grid((unsigned)cdiv(N, 1024), (unsigned)std::min(Tn - t0, 65535LL));
        hipLaunchKernelGGL((moe_join_kernel<T>), grid, dim3(256), 0, stream, y + t0 * S * ld, ld, ids + t0 * S, weights + t0 * S, S, E, N, C + t0 * ldct, ldct);
    }
    G9_HIP(hipGetLastError());
    return 0;
}

template <class T>
static int experts(int Tn, int S, const int *ids, const void *X, int64_t ldt, int64_t lds, const gen9blas_mx4 *W, const gen9blas_mx4 *gate,
                   const float *weights, void *C, int64_t ldct, int64_t ldcs) {
    const long long n = (long long)Tn * S;
    const int E = W->count, N = W->rows;
    // The rows of a tile, by places an expert: 64 go to the tile kernel, fewer to the kernels that read the weights once. µs with 16, 32
    // and 64, of 64 experts: FP16 gated 1536 × 4096, 6 places each 74.7, 75.9 and more, 8 81.9, 77.1 and 102, 32 149, 117 and 126, 48 200, 153
    // and 147; not gated 4096 × 1536, 6 48.7, 48.9, 8 53.9, 51.0 and 64, 32 106, 82 and 83, 48 148, 109 and 97. FP32, whose three pieces
    // of 32 rows LDS passes no faster than 16 twice: gated 32 208, 216 and 268, 64 364, 308 and 338; not gated 48 173, 185 and 181, 64 219,
    // 215 and 206.
    constexpr bool F = sizeof(T) == 4;
    const int rows = n > FEW_PLACES && n > (F ? 56LL : 40LL) * E ? 64 : !F && n >= 7LL * E ? 32 : 16;
    // Few places: each workgroup finds its rows among the ids itself (8 places 17.5 µs a call with a plan, whose kernel comes first)
    const bool direct = n <= FEW_PLACES;
    const long long most = direct ? n : cdiv(n, rows) + E + 1;
    if (n > 0x7fffffff) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "moe_gemm: T = %d tokens of S = %d places", Tn, S);
    void *plan = nullptr, *slots = nullptr;
    const long long ld = (N + 3) / 4 * 4LL;
    if (weights) G9_TRY(scratch(SLOT_SLOTS, (size_t)n * ld * 4, &slots));
    Rows R = {X, C, ldt, lds, ldct, ldcs, (int)n, S, nullptr, nullptr, nullptr, direct ? ids : nullptr};
    if (!direct) {
        G9_TRY(scratch(SLOT_PLAN, (size_t)(n + E + 3 + 2 * most) * 4, &plan));
        int *order = (int *)plan, *off = order + n, *tiles = off + E + 3;
        hipLaunchKernelGGL(moe_plan_kernel, dim3(1), dim3(1024), 0, stream, ids, (int)n, E, rows, order, off, tiles, (int)most);
        G9_HIP(hipGetLastError());
        R.tiles = tiles, R.order = order, R.off = off;
    }
    const Mx4View w = view(W), g = gate ? view(gate) : w;
    if (!weights)
        return gate ? launch_grouped<T, T, true>(R, w, g, E, (int)most, rows, Tn, n) : launch_grouped<T, T, false>(R, w, g, E, (int)most, rows, Tn, n);
    R.C = slots, R.ldct = S * ld, R.ldcs = ld;
    G9_TRY((gate ? launch_grouped<T, float, true>(R, w, g, E, (int)most, rows, Tn, n) : launch_grouped<T, float, false>(R, w, g, E, (int)most, rows, Tn, n)));
    return join((const float *)slots, ld, ids, weights, Tn, S, E, N, (T *)C, ldct);
}

}  // namespace g9llm

using namespace g9llm;

extern "C" {

int gen9blas_moe_route(int type, int T, int E, const void *logits, int ldl, const float *bias, int score, int groups, int top_groups, int k,
                       int renorm, float scale, int *ids, float *weights) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "moe_route: type %d unavailable", type);
    if (score != GEN9BLAS_SOFTMAX && score != GEN9BLAS_SIGMOID) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "moe_route: score %d unavailable", score);
    if (E < 1 || E > MAX_EXPERTS || k < 1 || k > MAX_K || k > E || ldl < E)
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "moe_route: E = %d (1..%d), k = %d (1..min(E, %d)), ldl = %d", E, MAX_EXPERTS, k, MAX_K, ldl);
    if (groups < 1 || groups > 64 || E % groups || top_groups < 1 || top_groups > groups)
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "moe_route: groups = %d (1..64, a divisor of E = %d), top_groups = %d", groups, E, top_groups);
    if (T <= 0) return 0;
    G9_TRY(need_device(logits, ((size_t)(T - 1) * ldl + E) * elem_size(type), "moe_route: logits"));
    if (bias) G9_TRY(need_device(bias, (size_t)E * 4, "moe_route: bias"));
    G9_TRY(need_device(ids, (size_t)T * k * 4, "moe_route: ids"));
    G9_TRY(need_device(weights, (size_t)T * k * 4, "moe_route: weights"));
    const RouteArgs a = {logits, ldl, bias, T, E, score == GEN9BLAS_SIGMOID, groups, top_groups, k, renorm, scale, ids, weights};
    return type == GEN9BLAS_H ? launch_route<_Float16>(a) : launch_route<float>(a);
}

int gen9blas_moe_gemm(int type, int T, int S, const int *ids, const void *X, int64_t ldt, int64_t lds, const gen9blas_mx4 *W,
                      const gen9blas_mx4 *gate, const float *weights, void *C, int64_t ldct, int64_t ldcs) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "moe_gemm: type %d unavailable", type);
    if (!W || W->count > MAX_EXPERTS) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "moe_gemm: %s", W ? "more than 1024 experts" : "no W");
    if (gate && (gate->count != W->count || gate->rows != W->rows || gate->K != W->K))
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "moe_gemm: the gate's shape is not W's");
    if (T <= 0 || (S <= 0 && !weights)) return 0;
    const int K = W->K, N = W->rows, es = elem_size(type);
    if (S <= 0) {   // sums of nothing
        if (ldct < N) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "moe_gemm: rows of C overlap (ldct %lld, N %d)", (long long)ldct, N);
        G9_TRY(need_device(C, ((size_t)(T - 1) * ldct + N) * es, "moe_gemm: C"));
        return type == GEN9BLAS_H ? join(nullptr, 0, nullptr, nullptr, T, 0, 0, N, (_Float16 *)C, ldct) : join(nullptr, 0, nullptr, nullptr, T, 0, 0, N, (float *)C, ldct);
    }
    if (lds < 0 || (lds > 0 && lds < K) || ldt < (lds ? (S - 1) * lds + K : K))
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "moe_gemm: rows of X overlap (ldt %lld, lds %lld, K %d)", (long long)ldt, (long long)lds, K);
    if (weights ? ldct < N : (ldcs < N || ldct < (S - 1) * ldcs + N))
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "moe_gemm: rows of C overlap (ldct %lld, ldcs %lld, N %d)", (long long)ldct, (long long)ldcs, N);
    G9_TRY(need_device(ids, (size_t)T * S * 4, "moe_gemm: ids"));
    G9_TRY(need_device(X, ((size_t)(T - 1) * ldt + (size_t)(S - 1) * lds + K) * es, "moe_gemm: X"));
    G9_TRY(need_device(C, ((size_t)(T - 1) * ldct + (weights ? 0 : (size_t)(S - 1) * ldcs) + N) * es, "moe_gemm: C"));
    if (weights) G9_TRY(need_device(weights, (size_t)T * S * 4, "moe_gemm: weights"));
    return type == GEN9BLAS_H ? experts<_Float16>(T, S, ids, X, ldt, lds, W, gate, weights, C, ldct, ldcs)
                              : experts<float>(T, S, ids, X, ldt, lds, W, gate, weights, C, ldct, ldcs);
}

}  // extern "C"
