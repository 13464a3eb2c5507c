// Rows of a table by tokens (gen9blas_embedding), and the table's gradient (gen9blas_embedding_backward).
//
// The gradient of row v is the sum of the rows of dY whose token is v. The tokens are sorted (stably, so that each row's sum
// has the order of its tokens), and the sorted list is cut into pieces of equal length: a workgroup adds up what its piece
// has, stores the rows whose tokens all lie in it, and leaves the sums of the first and the last row, where their tokens go on in
// the pieces before or behind, to a second kernel. So a token as frequent as all others together costs no more than they do,
// no sum depends on the order in which workgroups run, and no atomics are needed. Rows without tokens are cleared by other
// workgroups of the same launch.
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

// ---- the sort: least digits first, 8 bits a pass ----
// A workgroup has `per` consecutive places (a multiple of 1024). The first pass reads the ids themselves; the last place of a list
// of n is n − 1.
struct Sorted { int *key, *at; };   // of the place: the row, and the token

__device__ __forceinline__ void place(const Ids &ids, const Sorted &in, long long i, int V, int &key, int &at) {
    if (in.key) key = in.key[i], at = in.at[i];
    else key = ids.key(i, V), at = (int)i;
}
// counts[workgroup][digit]; the first pass clears the marks of the rows that have tokens, too.
__global__ void __launch_bounds__(256) sort_count_kernel(Ids ids, Sorted in, int n, int V, int shift, int per, int *__restrict__ counts, uint8_t *__restrict__ has) {
    __shared__ int count[256];
    count[threadIdx.x] = 0;
    if (has)
        for (long long v = (long long)blockIdx.x * 256 + threadIdx.x; v < V; v += (long long)gridDim.x * 256) has[v] = 0;
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
// Within 1024 places, a wave counts its lanes of a digit by ballots, and the waves' counts are added in their order.
__global__ void __launch_bounds__(1024) sort_place_kernel(Ids ids, Sorted in, int n, int V, int shift, int per, const int *__restrict__ counts, Sorted out, uint8_t *__restrict__ has) {
    __shared__ int base[256], all[256], wave_count[16][256];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    if (t < 256) {
        int before = 0, total = 0;
        for (int b = 0; b < (int)gridDim.x; b++) {
            const int c = counts[b * 256 + t];
            if (b < (int)blockIdx.x) before += c;
            total += c;
        }
        base[t] = before, all[t] = total;
    }
    __syncthreads();
    for (int d = 1; d < 256; d <<= 1) {   // sums up to each digit
        const int v = t < 256 && t >= d ? all[t - d] : 0;
        __syncthreads();
        if (t < 256) all[t] += v;
        __syncthreads();
    }
    if (t > 0 && t < 256) base[t] += all[t - 1];
    const long long end = min((long long)n, (blockIdx.x + 1LL) * per);
    for (long long i0 = (long long)blockIdx.x * per; i0 < end; i0 += 1024) {
        for (int i = t; i < 16 * 256; i += 1024) (&wave_count[0][0])[i] = 0;
        __syncthreads();
        const long long i = i0 + t;
        const bool mine = i < end;
        int key = 0, at = 0;
        if (mine) place(ids, in, i, V, key, at);
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
            int at0 = base[t];
            for (int w = 0; w < 16; w++) {
                const int c = wave_count[w][t];
                wave_count[w][t] = at0;
                at0 += c;
            }
            base[t] = at0;
        }
        __syncthreads();
        if (mine) {
            const int to = wave_count[wv][digit] + rank;
            out.key[to] = key, out.at[to] = at;
            if (has && key < V) has[key] = 1;
        }
        __syncthreads();
    }
}

// ---- the sums ----
struct GradArgs {
    const void *dY;
    long long lddy;
    Sorted s;
    const uint8_t *has;   // null: rows without tokens stay
    void *out;
    long long ldo;
    float *parts;         // two rows of ldp for each piece
    long long ldp;
    float scale;
    int n, V, D, per, pieces, cols, accumulate;
};
template <class T, int E> __device__ __forceinline__ void put(const GradArgs &a, int key, int d, const float *sum) {
    T *o = (T *)a.out + key * a.ldo + d;
    float v[E];
    if (a.accumulate) load_some<E>(o, a.D - d, v);
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = a.accumulate ? __builtin_fmaf(sum[e], a.scale, v[e]) : sum[e] * a.scale;
    store_some<E>(o, a.D - d, v);
}
// 2^cols threads side by side have 8 columns each; blockIdx.x: pieces, then groups of 64 rows to clear; blockIdx.y: columns.
template <class T, class O>
__global__ void __launch_bounds__(256) embedding_grad_kernel(GradArgs a) {
    constexpr int E = 8;
    const int c = threadIdx.x & ((1 << a.cols) - 1), side = threadIdx.x >> a.cols, sides = 256 >> a.cols;
    const int d = ((blockIdx.y << a.cols) + c) * E;
    if (d >= a.D) return;
    const int piece_groups = (a.pieces + sides - 1) / sides;
    if ((int)blockIdx.x >= piece_groups) {
        const float none[E] = {};
        const int v0 = (blockIdx.x - piece_groups) * 64;
        for (int v = v0 + side; v < min(v0 + 64, a.V); v += sides)
            if (!a.has[v]) store_some<E>((O *)a.out + v * a.ldo + d, a.D - d, none);
        return;
    }
    const int piece = blockIdx.x * sides + side;
    if (piece >= a.pieces) return;
    const int i0 = piece * a.per, i1 = (int)min((long long)i0 + a.per, (long long)a.n);
    const int before = i0 ? a.s.key[i0 - 1] : -1, behind = i1 < a.n ? a.s.key[i1] : -1;
    float sum[E] = {};
    int first = i0;
    for (int i = i0; i < i1; i++) {
        const int key = a.s.key[i];
        if (key >= a.V) break;   // no row's: the end of the list
        float v[E];
        load_some<E>((const T *)a.dY + a.s.at[i] * a.lddy + d, a.D - d, v);
#pragma unroll
        for (int e = 0; e < E; e++) sum[e] += v[e];
        const int next = i + 1 < i1 ? a.s.key[i + 1] : behind;
        if (next == key && i + 1 < i1) continue;
        if ((first == i0 && before == key) || next == key) store_some<E>(a.parts + (2LL * piece + (first > i0)) * a.ldp + d, a.D - d, sum);
        else put<O, E>(a, key, d, sum);
#pragma unroll
        for (int e = 0; e < E; e++) sum[e] = 0.f;
        first = i + 1;
    }
}
// Rows whose tokens begin in a piece and go on in others.
template <class O>
__global__ void __launch_bounds__(256) embedding_join_kernel(GradArgs a) {
    constexpr int E = 8;
    const int c = threadIdx.x & ((1 << a.cols) - 1), side = threadIdx.x >> a.cols, sides = 256 >> a.cols;
    const int d = ((blockIdx.y << a.cols) + c) * E, piece = blockIdx.x * sides + side;
    if (d >= a.D || piece >= a.pieces - 1) return;
    const int i0 = piece * a.per, i1 = i0 + a.per, key = a.s.key[i1 - 1];
    if (key >= a.V || a.s.key[i1] != key) return;            // does not go on
    const bool whole = a.s.key[i0] == key;
    if (whole && i0 && a.s.key[i0 - 1] == key) return;       // begins in an earlier one
    float sum[E];
    load_some<E>(a.parts + (2LL * piece + !whole) * a.ldp + d, a.D - d, sum);
    for (int p = piece + 1; p < a.pieces && a.s.key[p * a.per] == key; p++) {
        float v[E];
        load_some<E>(a.parts + 2LL * p * a.ldp + d, a.D - d, v);
#pragma unroll
        for (int e = 0; e < E; e++) sum[e] += v[e];
    }
    put<O, E>(a, key, d, sum);
}

template <class T, class O>
static int gradient(int n, int V, int D, const T *dY, int lddy, const Ids &ids, float scale, O *out, int ldo, int accumulate) {
    // places of a workgroup of the sort, and of a piece: few enough of both that what reads all of them stays short
    const int per = (int)(cdiv(cdiv(n, 256), 1024) * 1024), groups = (int)cdiv(n, per);
    const int piece = (int)std::max(32LL, cdiv(n, 1024)), pieces = (int)cdiv(n, piece);
    const long long ldp = cdiv(D, 8) * 8;
    char *w;
    const size_t lists = (size_t)n * 4, marks = ((size_t)V + 15) / 16 * 16;
    G9_TRY(scratch(SLOT_SORT, 4 * lists + (size_t)groups * 1024 + marks, (void **)&w));
    Sorted s[2] = {{(int *)w, (int *)(w + lists)}, {(int *)(w + 2 * lists), (int *)(w + 3 * lists)}};
    int *counts = (int *)(w + 4 * lists);
    uint8_t *has = accumulate ? nullptr : (uint8_t *)(counts + groups * 256);
    Sorted in = {nullptr, nullptr};
    int bits = 1;
    while (bits < 31 && V >> bits) bits++;   // of V, which stands for no row
    for (int shift = 0, pass = 0; shift < bits; shift += 8, pass++) {
        uint8_t *h = pass ? nullptr : has;
        hipLaunchKernelGGL(sort_count_kernel, dim3(groups), dim3(256), 0, stream, ids, in, n, V, shift, per, counts, h);
        hipLaunchKernelGGL(sort_place_kernel, dim3(groups), dim3(1024), 0, stream, ids, in, n, V, shift, per, (const int *)counts, s[pass & 1], h);
        G9_HIP(hipGetLastError());
        in = s[pass & 1];
    }
    void *parts;
    G9_TRY(scratch(SLOT_SUMS, (size_t)pieces * 2 * ldp * 4, &parts));
    GradArgs a = {dY, lddy, in, has, out, ldo, (float *)parts, ldp, scale, n, V, D, piece, pieces, 0, accumulate};
    while (a.cols < 8 && (8 << a.cols) < D) a.cols++;
    const unsigned slabs = (unsigned)cdiv(D, 8 << a.cols), piece_groups = (unsigned)cdiv(pieces, 256 >> a.cols);
    if (slabs > 65535 || V > 1 << 29) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "embedding_backward: more rows or columns than one launch can index (V %d, D %d)", V, D);
    hipLaunchKernelGGL((embedding_grad_kernel<T, O>), dim3(piece_groups + (has ? (unsigned)cdiv(V, 64) : 0), slabs), dim3(256), 0, stream, a);
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
