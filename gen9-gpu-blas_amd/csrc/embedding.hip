// Rows of a table by tokens (gen9blas_embedding), and the table's gradient (gen9blas_embedding_backward).
//
// The gradient of row v is the sum of the rows of dY whose token is v. The tokens are sorted (stably, so that each row's sum
// has the order of its tokens), and the sorted list is cut into pieces of equal length: a workgroup adds up what its piece
// has, stores the rows whose tokens all lie in it, and leaves the sums of the first and the last row, where their tokens go on in
// the pieces before or behind, to a second kernel. So a token as frequent as all others together costs no more than they do,
// no sum depends on the order in which workgroups run, and no atomics are needed. Rows without tokens are cleared by other
// workgroups of these launches, beside the sort as well, which leaves most CUs idle.
//
// HBM bounds both. 16384 tokens, 32000 × 4096 FP16: 109 µs, of them 26 the sort's four launches, 77 the sums and the rest of the
// clearing, 7 the join; the 134 MB of dY and the 262 MB of the result are 66 at 6 TB/s.
#include "llm.h"
#include "rows.h"
#include <algorithm>

namespace g9llm {

struct Ids {
    const void *p;
    int wide;   // 64 bits each
    __device__ __forceinline__ long long operator[](long long i) const { return wide ? ((const long long *)p)[i] : ((const int *)p)[i]; }
    // no row's: V
    __device__ __forceinline__ int key(long long i, int V) const {
        const long long v = (*this)[i];
        return v >= 0 && v < V ? (int)v : V;
    }
};

// A thread takes 16 bytes of a row.
template <class T>
__global__ void __launch_bounds__(256) embedding_kernel(const T *__restrict__ table, long long ldt, Ids ids, int Tn, int V, int D, int chunks, float scale, T *__restrict__ Y, long long ldy) {
    constexpr int E = 16 / sizeof(T);
    const long long total = (long long)Tn * chunks;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long t = i / chunks;
        const int d = (int)(i % chunks) * E, v = ids.key(t, V);
        float x[E] = {};
        if (v < V) {
            load_some<E>(table + v * ldt + d, D - d, x);
#pragma unroll
            for (int e = 0; e < E; e++) x[e] *= scale;
        }
        store_some<E>(Y + t * ldy + d, D - d, x);
    }
}

// Rows without tokens are cleared in groups of CLEAR, whole rows, so that what is written at a time lies together.
constexpr int CLEAR = 16;
struct ClearArgs {
    const uint8_t *has;   // of each row whether it has tokens; null: clear all
    void *out;
    long long ldo;
    int V, D, groups, cols;   // 2^cols threads side by side
};
// Thread c of `threads`: whole 16 bytes at 16-byte addresses, past the caches, and single elements before and behind.
template <class O> __device__ __forceinline__ void clear_row(O *row, int D, int c, int threads) {
    constexpr int V = 16 / sizeof(O);
    typedef O Vec __attribute__((ext_vector_type(V)));
    const int head = min((int)(-(uintptr_t)row & 15) / (int)sizeof(O), D), body = (D - head) / V * V;
    for (int x = c; x < D - body; x += threads) row[x < head ? x : x + body] = O(0);
    for (int x = c * V; x < body; x += V * threads) __builtin_nontemporal_store(Vec{}, reinterpret_cast<Vec *>(row + head + x));
}
template <class O> __device__ __forceinline__ void clear_rows(const ClearArgs &a, long long group) {
    const long long v0 = group * CLEAR;
    const int lane = threadIdx.x & 63, c = threadIdx.x & ((1 << a.cols) - 1);
    const unsigned long long empty = __ballot(lane < CLEAR && v0 + lane < a.V && !(a.has && a.has[min(v0 + lane, a.V - 1LL)]));
    for (int r = threadIdx.x >> a.cols; r < CLEAR; r += (int)blockDim.x >> a.cols) {
        if (!(empty >> r & 1)) continue;
        clear_row((O *)a.out + (v0 + r) * a.ldo, a.D, c, 1 << a.cols);
    }
}

// ---- the sort: least digits first, 8 bits a pass ----
// A workgroup has `per` consecutive places (a multiple of 1024). The first pass reads the ids themselves; the last place of a list
// of n is n − 1.
struct Sorted { int *key, *at; };   // of the place: the row, and the token

__device__ __forceinline__ void place(const Ids &ids, const Sorted &in, long long i, int V, int &key, int &at) {
    if (in.key) key = in.key[i], at = in.at[i];
    else key = ids.key(i, V), at = (int)i;
}
// counts[workgroup][digit]; the first pass clears the marks of the rows that have tokens, too. Workgroups behind the `groups` of the
// sort, which leave most CUs idle, clear rows from group `first` on: in the first pass, whose marks are not set yet, all of them (the
// sums come later), then those without tokens.
template <class O>
__global__ void __launch_bounds__(256) sort_count_kernel(Ids ids, Sorted in, int n, int V, int shift, int per, int *__restrict__ counts, uint8_t *__restrict__ has, int groups, ClearArgs clear, int first) {
    if ((int)blockIdx.x >= groups) {
        clear_rows<O>(clear, first + blockIdx.x - groups);
        return;
    }
    __shared__ int count[256];
    count[threadIdx.x] = 0;
    if (has)
        for (long long v = (long long)blockIdx.x * 256 + threadIdx.x; v < V; v += (long long)groups * 256) has[v] = 0;
    __syncthreads();
    const long long end = min((long long)n, (blockIdx.x + 1LL) * per);
    for (long long i = (long long)blockIdx.x * per + threadIdx.x; i < end; i += 256) {
        const int key = in.key ? in.key[i] : ids.key(i, V);
        atomicAdd(&count[key >> shift & 255], 1);
    }
    __syncthreads();
    counts[blockIdx.x * 256 + threadIdx.x] = count[threadIdx.x];
}
// Where a workgroup's places of a digit begin: all places of smaller digits, and this digit's of the workgroups before.
// Within 1024 places, a wave counts its lanes of a digit by ballots, and the waves' counts are added in their order. Latencies bound
// it: 16384 tokens 6 µs a pass (9 with the sums over digits by barriers, and the waves' counts read one after the other).
template <class O>
__global__ void __launch_bounds__(1024) sort_place_kernel(Ids ids, Sorted in, int n, int V, int shift, int per, const int *__restrict__ counts, Sorted out, uint8_t *__restrict__ has, int groups, ClearArgs clear, int from) {
    if ((int)blockIdx.x >= groups) {
        clear_rows<O>(clear, from + blockIdx.x - groups);
        return;
    }
    __shared__ int waves[4], wave_count[16][256];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const long long begin = (long long)blockIdx.x * per, end = min((long long)n, begin + per);
    int key = 0, at = 0;
    if (begin + t < end) place(ids, in, begin + t, V, key, at);   // on its way while the places are found
    for (int i = t; i < 16 * 256; i += 1024) (&wave_count[0][0])[i] = 0;
    int base = 0;   // threads 0..255: of the digit with this number
    if (t < 256) {
        int before = 0, total = 0;
#pragma unroll 8
        for (int b = 0; b < groups; b++) {
            const int c = counts[b * 256 + t];
            before += b < (int)blockIdx.x ? c : 0;
            total += c;
        }
        int sum = total;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(sum, d);
            if (lane >= d) sum += v;
        }
        if (lane == 63) waves[wv] = sum;
        base = before + sum - total;
    }
    __syncthreads();
    if (t < 256)
        for (int w = 0; w < wv; w++) base += waves[w];
    for (long long i0 = begin; i0 < end; i0 += 1024) {
        const long long i = i0 + t;
        const bool mine = i < end;
        const int digit = key >> shift & 255;
        unsigned long long same = __ballot(mine);
#pragma unroll
        for (int b = 0; b < 8; b++) {
            const bool bit = digit >> b & 1;
            const unsigned long long set = __ballot(bit);
            same &= bit ? set : ~set;
        }
        const int rank = __popcll(same & ((1ULL << lane) - 1));
        if (mine && rank == 0) wave_count[wv][digit] = __popcll(same);
        __syncthreads();
        if (t < 256) {
            int c[16];
#pragma unroll
            for (int w = 0; w < 16; w++) c[w] = wave_count[w][t];
#pragma unroll
            for (int w = 0; w < 16; w++) {
                wave_count[w][t] = base;
                base += c[w];
            }
        }
        __syncthreads();
        if (mine) {
            const int to = wave_count[wv][digit] + rank;
            out.key[to] = key, out.at[to] = at;
            if (has && key < V) has[key] = 1;
        }
        if (i0 + 1024 >= end) break;
        if (i + 1024 < end) place(ids, in, i + 1024, V, key, at);
        __syncthreads();
        for (int j = t; j < 16 * 256; j += 1024) (&wave_count[0][0])[j] = 0;
        __syncthreads();
    }
}

// Up to 4096 tokens: the whole sort in one workgroup, in LDS (2000 tokens 9 µs, 4000 16).
constexpr int SMALL = 4096;
__global__ void __launch_bounds__(1024) sort_small_kernel(Ids ids, int n, int V, int bits, Sorted out, uint8_t *__restrict__ has) {
    __shared__ int keys[2][SMALL], ats[2][SMALL], waves[4], wave_count[16][256], base[256];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    if (has)
        for (int v = t * 16; v < V; v += 1024 * 16) *reinterpret_cast<u32x4 *>(has + v) = u32x4{0, 0, 0, 0};   // rounded up to 16
    __syncthreads();
    for (int i = t; i < n; i += 1024) {
        const int key = ids.key(i, V);
        keys[0][i] = key, ats[0][i] = i;
        if (has && key < V) has[key] = 1;
    }
    int from = 0;
    for (int shift = 0; shift < bits; shift += 8, from ^= 1) {
        if (t < 256) base[t] = 0;
        __syncthreads();
        for (int i = t; i < n; i += 1024) atomicAdd(&base[keys[from][i] >> shift & 255], 1);
        __syncthreads();
        int mine = 0, sum = 0;
        if (t < 256) {
            mine = sum = base[t];
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int v = __shfl_up(sum, d);
                if (lane >= d) sum += v;
            }
            if (lane == 63) waves[wv] = sum;
        }
        __syncthreads();
        if (t < 256) {
            sum -= mine;
            for (int w = 0; w < wv; w++) sum += waves[w];
        }
        for (int i0 = 0; i0 < n; i0 += 1024) {
            for (int j = t; j < 16 * 256; j += 1024) (&wave_count[0][0])[j] = 0;
            __syncthreads();
            const int i = i0 + t;
            const bool is = i < n;
            const int key = is ? keys[from][i] : 0, digit = key >> shift & 255;
            unsigned long long same = __ballot(is);
#pragma unroll
            for (int b = 0; b < 8; b++) {
                const bool bit = digit >> b & 1;
                const unsigned long long set = __ballot(bit);
                same &= bit ? set : ~set;
            }
            const int rank = __popcll(same & ((1ULL << lane) - 1));
            if (is && rank == 0) wave_count[wv][digit] = __popcll(same);
            __syncthreads();
            if (t < 256) {
                int c[16];
#pragma unroll
                for (int w = 0; w < 16; w++) c[w] = wave_count[w][t];
#pragma unroll
                for (int w = 0; w < 16; w++) {
                    wave_count[w][t] = sum;
                    sum += c[w];
                }
            }
            __syncthreads();
            if (is) {
                const int to = wave_count[wv][digit] + rank;
                keys[from ^ 1][to] = key, ats[from ^ 1][to] = ats[from][i];
            }
            __syncthreads();
        }
    }
    for (int i = t; i < n; i += 1024) out.key[i] = keys[from][i], out.at[i] = ats[from][i];
}

// ---- the sums ----
struct GradArgs {
    const void *dY;
    long long lddy;
    Sorted s;
    void *out;
    long long ldo;
    float *parts;         // two rows of ldp for each piece
    long long ldp;
    float scale;
    int n, V, D, per, pieces, cols, accumulate;
    int past;             // results go out past the caches: FP16 rows of whole 128-byte lines
};
template <class T, int E> __device__ __forceinline__ void put(const GradArgs &a, int key, int d, const float *sum) {
    T *o = (T *)a.out + key * a.ldo + d;
    float v[E];
    if (a.accumulate) load_some<E>(o, a.D - d, v);
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = a.accumulate ? __builtin_fmaf(sum[e], a.scale, v[e]) : sum[e] * a.scale;
    if (a.past) store_some<E, T, true>(o, a.D - d, v);
    else store_some<E>(o, a.D - d, v);
}
// 2^cols threads side by side have 8 columns each; blockIdx.x: pieces (blockIdx.y: their columns), then groups of rows to clear.
template <class T, class O>
__global__ void __launch_bounds__(256) embedding_grad_kernel(GradArgs a, ClearArgs clear, int cleared) {
    constexpr int E = 8, U = 8;
    const int c = threadIdx.x & ((1 << a.cols) - 1), side = threadIdx.x >> a.cols, sides = 256 >> a.cols;
    const int d = ((blockIdx.y << a.cols) + c) * E;
    const int piece_groups = (a.pieces + sides - 1) / sides;
    if ((int)blockIdx.x >= piece_groups) {
        clear_rows<O>(clear, cleared + (long long)(blockIdx.x - piece_groups) * gridDim.y + blockIdx.y);
        return;
    }
    if (d >= a.D) return;
    const int piece = blockIdx.x * sides + side;
    if (piece >= a.pieces) return;
    const int i0 = piece * a.per, i1 = (int)min((long long)i0 + a.per, (long long)a.n);
    const int before = i0 ? a.s.key[i0 - 1] : -1, behind = i1 < a.n ? a.s.key[i1] : -1;
    float sum[E] = {};
    int first = i0;
    for (int i = i0; i < i1; i += U) {   // U rows on their way
        int key[U + 1];
        float v[U][E];
#pragma unroll
        for (int u = 0; u <= U; u++) key[u] = i + u < i1 ? a.s.key[i + u] : behind;
#pragma unroll
        for (int u = 0; u < U; u++) load_some<E>((const T *)a.dY + a.s.at[min(i + u, i1 - 1)] * a.lddy + d, a.D - d, v[u]);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + u >= i1 || key[u] >= a.V) return;   // no row's: the end of the list
#pragma unroll
            for (int e = 0; e < E; e++) sum[e] += v[u][e];
            if (key[u + 1] == key[u] && i + u + 1 < i1) continue;
            if ((first == i0 && before == key[u]) || key[u + 1] == key[u]) store_some<E>(a.parts + (2LL * piece + (first > i0)) * a.ldp + d, a.D - d, sum);
            else put<O, E>(a, key[u], d, sum);
#pragma unroll
            for (int e = 0; e < E; e++) sum[e] = 0.f;
            first = i + u + 1;
        }
    }
}
// Rows whose tokens begin in a piece and go on in others.
template <class O>
__global__ void __launch_bounds__(256) embedding_join_kernel(GradArgs a) {
    constexpr int E = 8, U = 8;
    const int c = threadIdx.x & ((1 << a.cols) - 1), side = threadIdx.x >> a.cols, sides = 256 >> a.cols;
    const int d = ((blockIdx.y << a.cols) + c) * E, piece = blockIdx.x * sides + side;
    if (d >= a.D || piece >= a.pieces - 1) return;
    const int i0 = piece * a.per, i1 = i0 + a.per, key = a.s.key[i1 - 1], behind = a.s.key[i1], first = a.s.key[i0], before = i0 ? a.s.key[i0 - 1] : -1;
    const bool whole = first == key;
    if (key >= a.V || behind != key || (whole && before == key)) return;   // does not go on, or begins in an earlier one
    float sum[E];
    load_some<E>(a.parts + (2LL * piece + !whole) * a.ldp + d, a.D - d, sum);
    for (int p = piece + 1; p < a.pieces; p += U) {
        int at[U];
        float v[U][E];
#pragma unroll
        for (int u = 0; u < U; u++) at[u] = a.s.key[min(p + u, a.pieces - 1) * a.per];
        int more = 0;   // pieces that go on with this row, of the next U
#pragma unroll
        for (int u = 0; u < U; u++) more += p + u < a.pieces && at[u] == key;
#pragma unroll
        for (int u = 0; u < U; u++)
            if (u < more) load_some<E>(a.parts + 2LL * (p + u) * a.ldp + d, a.D - d, v[u]);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (u < more)
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] += v[u][e];
        if (more < U) break;
    }
    put<O, E>(a, key, d, sum);
}

// Up to 1024 tokens in one launch, without work buffers: a workgroup has `rows` rows and 8 << cols columns. It sorts the tokens of
// its rows by row in LDS, each wave a quarter of them in their order, cuts that list into a piece for each of its 256 >> cols rows
// of threads, and joins the pieces' ends through LDS: as the kernels above do through memory. The rows without tokens are
// dealt out among the workgroups of the same rows. The read of the tokens' first rows bounds it (1976 × 152 FP32, 64 tokens 6 µs), or
// the clearing does (32000 × 4096 FP16 56).
constexpr int FEW = 1024;
template <class T, class O>
__global__ void __launch_bounds__(256) embedding_few_kernel(GradArgs a, Ids ids, int rows, int clear_cols) {
    constexpr int E = 8, U = 8;
    __shared__ int list[FEW], base[4][64], total;   // list: row << 16 | token
    __shared__ unsigned long long none;
    __shared__ float part[256][2][E];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int v0 = blockIdx.x * rows, mine = min(rows, a.V - v0);
    const int quarter = (a.n + 3) / 4, t0 = wv * quarter, t1 = min(t0 + quarter, a.n);
    base[wv][lane] = 0;
    __syncthreads();
    for (int i = t0 + lane; i < t1; i += 64) {
        const int r = ids.key(i, a.V) - v0;   // no row's: V − v0 >= mine
        if (r >= 0 && r < mine) atomicAdd(&base[wv][r], 1);
    }
    __syncthreads();
    if (wv == 0) {   // a lane a row: where each wave's tokens of it begin
        int c[4], sum = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) c[w] = base[w][lane], sum += c[w];
        int end = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(end, d);
            if (lane >= d) end += v;
        }
        int at = end - sum;
#pragma unroll
        for (int w = 0; w < 4; w++) base[w][lane] = at, at += c[w];
        const unsigned long long empty = __ballot(sum == 0 && lane < mine);
        if (lane == 63) total = end, none = empty;
    }
    __syncthreads();
    const int m = total;
    if (!a.accumulate) {
        const unsigned long long empty = none;
        const int c = t & ((1 << clear_cols) - 1);
        for (int r = blockIdx.y + (t >> clear_cols) * gridDim.y; r < mine; r += (256 >> clear_cols) * gridDim.y)
            if (empty >> r & 1) clear_row((O *)a.out + (long long)(v0 + r) * a.ldo, a.D, c, 1 << clear_cols);
    }
    if (!m) return;
    for (int i0 = t0; i0 < t1; i0 += 64) {
        const int i = i0 + lane, r = i < t1 ? ids.key(i, a.V) - v0 : -1;
        const bool is = r >= 0 && r < mine;
        unsigned long long same = __ballot(is);
        if (!same) continue;
#pragma unroll
        for (int b = 0; b < 6; b++) {
            const bool bit = r >> b & 1;
            const unsigned long long set = __ballot(bit);
            same &= bit ? set : ~set;
        }
        const int rank = __popcll(same & ((1ULL << lane) - 1)), at = is ? base[wv][r] : 0;
        __builtin_amdgcn_wave_barrier();
        if (is) {
            list[at + rank] = r << 16 | i;
            if (rank == 0) base[wv][r] = at + __popcll(same);
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    const int c = t & ((1 << a.cols) - 1), side = t >> a.cols, d = ((blockIdx.y << a.cols) + c) * E;
    const int per = (m + (256 >> a.cols) - 1) / (256 >> a.cols), i0 = min(side * per, m), i1 = d < a.D ? min(i0 + per, m) : i0;
    auto row = [&](int i) { return list[i] >> 16; };
    float sum[E] = {};
    if (i0 < i1) {
        const int before = i0 ? row(i0 - 1) : -1, behind = i1 < m ? row(i1) : -1;
        int first = i0;
        for (int i = i0; i < i1; i += U) {   // U rows on their way
            float v[U][E];
#pragma unroll
            for (int u = 0; u < U; u++) load_some<E>((const T *)a.dY + (list[min(i + u, i1 - 1)] & 0xffff) * a.lddy + d, a.D - d, v[u]);
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (i + u >= i1) break;
                const int key = row(i + u), next = i + u + 1 < i1 ? row(i + u + 1) : behind;
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] += v[u][e];
                if (next == key && i + u + 1 < i1) continue;
                if ((first == i0 && before == key) || next == key) {
#pragma unroll
                    for (int e = 0; e < E; e++) part[t][first > i0][e] = sum[e];
                } else put<O, E>(a, v0 + key, d, sum);
#pragma unroll
                for (int e = 0; e < E; e++) sum[e] = 0.f;
                first = i + u + 1;
            }
        }
    }
    __syncthreads();
    if (i0 >= i1 || i1 == m) return;
    const int key = row(i1 - 1);
    const bool whole = row(i0) == key;
    if (row(i1) != key || (whole && i0 && row(i0 - 1) == key)) return;   // does not go on, or begins in an earlier one
#pragma unroll
    for (int e = 0; e < E; e++) sum[e] = part[t][!whole][e];
    for (int p = 1; i0 + p * per < m && row(i0 + p * per) == key; p++)
#pragma unroll
        for (int e = 0; e < E; e++) sum[e] += part[t + (p << a.cols)][0][e];
    put<O, E>(a, v0 + key, d, sum);
}

// The exponent of 2 of how many threads side by side, of 8 columns each, D columns take.
static int widths(int D, int most) {
    int cols = 0;
    while (cols < most && (8 << cols) < D) cols++;
    return cols;
}
template <class T, class O>
static int gradient(int n, int V, int D, const T *dY, int lddy, const Ids &ids, float scale, O *out, int ldo, int accumulate) {
    const int past = sizeof(O) == 2 && (uintptr_t)out % 128 == 0 && ldo % 64 == 0;
    const int cols = widths(D, 8);
    // Few tokens: every workgroup reads all of them, so the columns of one, which narrow leave more threads for a token's sum, are as wide
    // as 10 workgroups a CU ask for; and with nothing to clear, 20 a CU are the most (µs, here / sorted by a launch of its own: 816 tokens,
    // 1976 × 152 FP32 7.6 / 15.6, one token in all places 15 / 30; 32000 × 1024 FP16 20 / 23, one token 45 / 39; 32000 × 4096 FP32 101 /
    // 111; 256 tokens accumulated, 32000 × 4096 19 / 15, 64 tokens 14 / 16).
    int few_cols = std::min(cols, 3);
    auto workgroups = [&](int rows) { return cdiv(V, rows) * cdiv(D, 8 << few_cols); };
    while (few_cols < std::min(cols, 5) && workgroups(64) > 10 * num_cus) few_cols++;
    if (n <= FEW && D <= 1 << 21 && V <= 1 << 27 && (!accumulate || n <= 64 || workgroups(64) <= 20 * num_cus)) {
        const int rows = workgroups(64) >= 2 * num_cus ? 64 : 16;
        const GradArgs a = {dY, lddy, {}, out, ldo, nullptr, 0, scale, n, V, D, 0, 0, few_cols, accumulate, past};
        hipLaunchKernelGGL((embedding_few_kernel<T, O>), dim3((unsigned)cdiv(V, rows), (unsigned)cdiv(D, 8 << few_cols)), dim3(256), 0, stream, a, ids, rows, cols);
        G9_HIP(hipGetLastError());
        return 0;
    }
    // places of a workgroup of the sort, and of a piece: few enough of both that what reads all of them stays short
    const int per = (int)(cdiv(cdiv(n, 256), 1024) * 1024), groups = (int)cdiv(n, per);
    const int piece = (int)std::max(8LL, cdiv(n, 512)), pieces = (int)cdiv(n, piece);
    const long long ldp = cdiv(D, 8) * 8;
    const unsigned slabs = (unsigned)cdiv(D, 8 << cols), piece_groups = (unsigned)cdiv(pieces, 256 >> cols);
    if (slabs > 65535 || V > 1 << 27 || n > 0x7ffff000) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "embedding_backward: more than kernels can index (%d tokens, V %d, D %d)", n, V, D);
    char *w;
    const size_t lists = ((size_t)n * 4 + 15) / 16 * 16, marks = ((size_t)V + 15) / 16 * 16;
    G9_TRY(work_buffer("embedding_backward", SLOT_SORT, 4 * lists + (size_t)groups * 1024 + marks, (void **)&w));
    Sorted s[2] = {{(int *)w, (int *)(w + lists)}, {(int *)(w + 2 * lists), (int *)(w + 3 * lists)}};
    int *counts = (int *)(w + 4 * lists);
    uint8_t *has = accumulate ? nullptr : (uint8_t *)(counts + groups * 256);
    void *parts;
    G9_TRY(work_buffer("embedding_backward", SLOT_SUMS, (size_t)pieces * 2 * ldp * 4, &parts));

    const ClearArgs all = {has, out, ldo, V, D, has ? (int)cdiv(V, CLEAR) : 0, cols};
    int cleared = 0;   // groups of rows that the sort's launches have cleared
    int bits = 1;
    while (bits < 31 && V >> bits) bits++;   // of V, which stands for no row
    Sorted in = {nullptr, nullptr};
    // one workgroup clears a million marks in some 10 µs
    if (n <= SMALL && (!has || V <= 1 << 20)) {
        in = s[0];
        hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(1024), 0, stream, ids, n, V, bits, in, has);
    } else {
        // what the idle CUs clear beside a launch of the sort: about 4 µs of writing, 24 MB
        const int beside = (int)std::max<long long>(1, (24 << 20) / ((long long)CLEAR * D * (int)sizeof(O)));
        for (int shift = 0, pass = 0; shift < bits; shift += 8, pass++) {
            uint8_t *h = pass ? nullptr : has;
            ClearArgs clear = all;
            if (!pass) clear.has = nullptr;
            int more = std::min(beside, clear.groups - cleared);
            hipLaunchKernelGGL((sort_count_kernel<O>), dim3(groups + more), dim3(256), 0, stream, ids, in, n, V, shift, per, counts, h, groups, clear, cleared);
            cleared += more;
            more = std::min(beside, clear.groups - cleared);
            hipLaunchKernelGGL((sort_place_kernel<O>), dim3(groups + more), dim3(1024), 0, stream, ids, in, n, V, shift, per, (const int *)counts, s[pass & 1], h, groups, clear, cleared);
            cleared += more;
            in = s[pass & 1];
        }
    }
    G9_HIP(hipGetLastError());
    const GradArgs a = {dY, lddy, in, out, ldo, (float *)parts, ldp, scale, n, V, D, piece, pieces, cols, accumulate,
                        past};
    hipLaunchKernelGGL((embedding_grad_kernel<T, O>), dim3(piece_groups + (unsigned)cdiv(all.groups - cleared, slabs), slabs), dim3(256), 0, stream, a, all, cleared);
    G9_HIP(hipGetLastError());
    if (pieces > 1) hipLaunchKernelGGL((embedding_join_kernel<O>), dim3(piece_groups, slabs), dim3(256), 0, stream, a);
    G9_HIP(hipGetLastError());
    return 0;
}

// Clears rows of 2-byte words.
__global__ void __launch_bounds__(256) zero_rows_kernel(uint16_t *p, long long ld, long long words, long long total) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) p[i / words * ld + i % words] = 0;
}
int zero_rows(void *p, long long ld, long long rows, long long bytes) {
    const long long total = rows * (bytes / 2);
    if (total <= 0) return 0;
    hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)std::min(cdiv(total, 256), 16384LL)), dim3(256), 0, stream, (uint16_t *)p, ld / 2, bytes / 2, total);
    G9_HIP(hipGetLastError());
    return 0;
}

}  // namespace g9llm

using namespace g9llm;

extern "C" {

int gen9blas_embedding(int type, int T, int V, int D, const void *table, int ldt, const void *ids, int id_bytes, float scale, void *Y, int ldy) {
    G9_TRY(begin());
    if (type != GEN9BLAS_H && type != GEN9BLAS_S) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "embedding: type %d unavailable", type);
    if (id_bytes != 4 && id_bytes != 8) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "embedding: ids of %d bytes", id_bytes);
    if (T <= 0 || D <= 0) return 0;
    if (V < 1 || ldt < D || ldy < D) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "embedding: V %d, D %d, ldt %d, ldy %d", V, D, ldt, ldy);
    const size_t es = elem_size(type);
    G9_TRY(need_device(table, ((size_t)(V - 1) * ldt + D) * es, "embedding: table"));
    G9_TRY(need_device(ids, (size_t)T * id_bytes, "embedding: ids"));
    G9_TRY(need_device(Y, ((size_t)(T - 1) * ldy + D) * es, "embedding: Y"));
    const Ids i = {ids, id_bytes == 8};
    const int chunks = (int)cdiv(D, 16 / (int)es);
    const dim3 grid((unsigned)std::min(cdiv((long long)T * chunks, 256), 16384LL));
    if (type == GEN9BLAS_H) hipLaunchKernelGGL((embedding_kernel<_Float16>), grid, dim3(256), 0, stream, (const _Float16 *)table, ldt, i, T, V, D, chunks, scale, (_Float16 *)Y, ldy);
    else hipLaunchKernelGGL((embedding_kernel<float>), grid, dim3(256), 0, stream, (const float *)table, ldt, i, T, V, D, chunks, scale, (float *)Y, ldy);
    G9_HIP(hipGetLastError());
    return 0;
}

int gen9blas_embedding_backward(int type, int T, int V, int D, const void *dY, int lddy, const void *ids, int id_bytes, float scale, int out_type, void *dT, int lddt,
                                int accumulate) {
    G9_TRY(begin());
    if ((type != GEN9BLAS_H && type != GEN9BLAS_S) || (out_type != type && out_type != GEN9BLAS_S))
        G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "embedding_backward: types %d and %d unavailable", type, out_type);
    if (id_bytes != 4 && id_bytes != 8) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "embedding_backward: ids of %d bytes", id_bytes);
    if (V <= 0 || D <= 0) return 0;
    T = std::max(T, 0);
    if (lddy < D || lddt < D) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "embedding_backward: V %d, D %d, lddy %d, lddt %d", V, D, lddy, lddt);
    const size_t es = elem_size(type), os = elem_size(out_type);
    if (T) {
        G9_TRY(need_device(dY, ((size_t)(T - 1) * lddy + D) * es, "embedding_backward: dY"));
        G9_TRY(need_device(ids, (size_t)T * id_bytes, "embedding_backward: ids"));
    }
    G9_TRY(need_device(dT, ((size_t)(V - 1) * lddt + D) * os, "embedding_backward: dT"));
    if (!T) return accumulate ? 0 : zero_rows(dT, (long long)(lddt * os), V, (long long)(D * os));
    const Ids i = {ids, id_bytes == 8};
    typedef _Float16 H;
    if (type == GEN9BLAS_S) return gradient(T, V, D, (const float *)dY, lddy, i, scale, (float *)dT, lddt, accumulate);
    if (out_type == GEN9BLAS_S) return gradient(T, V, D, (const H *)dY, lddy, i, scale, (float *)dT, lddt, accumulate);
    return gradient(T, V, D, (const H *)dY, lddy, i, scale, (H *)dT, lddt, accumulate);
}

}  // extern "C"
