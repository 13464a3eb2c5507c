// Linear layers of a few dozen rows: the weights streamed once from memory.
//
// A workgroup has 64 columns, all rows (MT tiles of 16) and a slice of k, which goes through a ring of NS stages of 512 bytes of
// each row. Its eight waves are four groups of 16 columns, two waves each, which share the k of a stage, so that one's products
// run while the other waits for LDS. All copy their share of W and X into LDS (lds_dma16, two rows each). Chunk c (16 bytes) of row r
// lies at c ^ (r & 15), so that the 16 lanes that read one chunk of 16 rows do so from different banks. Lane 16g + r reads 16
// bytes of row r of W and of X, which is an operand of v_mfma_f32_16x16x32_f16 as it lies, and element s of four
// v_mfma_f32_16x16x4_f32 (a sum over k in any order). FP32 sums of a stage begin at zero and are added to the running ones, whose
// rounding grows with the stages then (24 × 4096 × 11008: 1.3e-7 of the result, one running sum 8e-7).
// One barrier a stage: behind it stage j is there, and stage j − 1 has been read and is filled again.
// 24 × 4096 × 11008 FP32 44 µs, 39 of them this kernel: 180 MB at 4.6 TB/s, what its 1.4 µs a stage leave of HBM's 6. The 64 × 64 tiles of
// the large products take 77, with 32 × 128 tiles 50. Operands straight from memory into registers 84 (a load of 16 bytes from each of 16 rows
// takes 80 clocks); four waves 55; pieces of k dealt out evenly over the CUs whatever the shape, with cut tiles, 53.
#pragma once
#include "linear_epilogue.h"
#include "lds_dma.h"

namespace g9llm {

template <class T> struct RowsArgs {
    const T *X, *W;
    T *Y;
    long long ldx, ldw, ldy;
    int M, N, K, slices, per;   // per: pieces of 512 bytes of k in a slice
    f32x4 *parts;               // slices > 1: their sums
    Epilogue<T> epilogue;
};

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <class T> __device__ __forceinline__ void rows_product(u32x4 w, u32x4 x, f32x4 &c) {
    if constexpr (sizeof(T) == 2) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), c, 0, 0, 0);
    } else {
        const f32x4 a = __builtin_bit_cast(f32x4, w), b = __builtin_bit_cast(f32x4, x);
#pragma unroll
        for (int s = 0; s < 4; s++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    }
}
template <class T> __device__ __forceinline__ void rows_store(const RowsArgs<T> &a, int tile, int wave, int j, int lane, f32x4 sum) {
    const int m = 16 * j + (lane & 15), n = tile * 64 + wave * 16 + 4 * (lane >> 4), valid = a.N - n;
    if (m >= a.M) return;
    a.epilogue.each([&](auto kind) {
        a.epilogue.template row<T, 4>(kind, a.Y, a.ldy, m, n, a.epilogue.template columns<4>(n, valid), a.epilogue.template residual<4>(m, a.M, n, valid), valid, sum);
    });
}

template <class T, int MT, int NS>
__global__ void __launch_bounds__(512) linear_rows_kernel(RowsArgs<T> a) {
    constexpr int V = 16 / sizeof(T), GK = 512 / sizeof(T);
    constexpr int WB = 64 * 512, SB = WB + MT * 16 * 512, LPS = 4 + MT;
    static_assert((NS - 1) * LPS < 64 && NS * SB <= 160 * 1024);
    __shared__ __attribute__((aligned(1024))) unsigned char smem[NS * SB];
    G9_LDS unsigned char *lds = (G9_LDS unsigned char *)smem;
    const unsigned base = (unsigned)(uintptr_t)lds;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, r16 = lane & 15;
    const int cols = wv & 3, half = wv >> 2;   // which 16 columns, and which half of a stage's k
    const int tile = blockIdx.x / a.slices, slice = blockIdx.x % a.slices, n0 = tile * 64;
    const int whole = a.K / GK, first = min(slice * a.per, whole), ng = min(whole - first, a.per);

    // copy i of a wave: rows 2i and 2i + 1 of its 8 of W, or of its 2·MT of X; lane l: row l / 32 of the two, position l % 32. Rows past
    // the last one are copies of it, whose sums nobody stores.
    const int sub = lane >> 5, pos = lane & 31;
    const char *wb = (const char *)(a.W + (long long)n0 * a.ldw), *xb = (const char *)a.X;
    unsigned woff[4], xoff[MT];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = wv * 8 + 2 * i + sub;
        woff[i] = (unsigned)(min(r, a.N - 1 - n0) * a.ldw * (long long)sizeof(T)) + ((pos ^ (r & 15)) << 4);
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int r = wv * 2 * MT + 2 * i + sub;
        xoff[i] = (unsigned)(min(r, a.M - 1) * a.ldx * (long long)sizeof(T)) + ((pos ^ (r & 15)) << 4);
    }
    // Workgroups of one slice read the same lines of X: in each XCD they begin at different ones (32 × 11008 × 4096 FP16 20.6 µs,
    // all at the first 23.8)
    const int rot = ng > 1 ? (int)((blockIdx.x >> 3) % (unsigned)ng) : 0;
    auto issue = [&](int j, int st) {   // past the last piece: the last one again, into a stage that nobody reads
        const int at = min(j, ng - 1) + rot;
        const long long k = (long long)(first + (at < ng ? at : at - ng)) * 512;
        const unsigned dst = base + st * SB;
#pragma unroll
        for (int i = 0; i < 4; i++) g9::lds_dma16(wb + k, woff[i], dst + (wv * 4 + i) * 1024);
#pragma unroll
        for (int i = 0; i < MT; i++) g9::lds_dma16(xb + k, xoff[i], dst + WB + (wv * MT + i) * 1024);
    };
    f32x4 acc[MT] = {};
    auto products = [&](const G9_LDS unsigned char *s) {
        constexpr int SUMS = sizeof(T) == 4 ? 2 : 1;   // FP32: of the even and the odd chunks
        f32x4 sum[SUMS][MT] = {};
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int at = r16 * 512 + (((16 * half + 4 * t + g) ^ r16) << 4);
            const u32x4 w = *reinterpret_cast<const G9_LDS u32x4 *>(s + cols * 8192 + at);
#pragma unroll
            for (int j = 0; j < MT; j++) {
                const u32x4 x = *reinterpret_cast<const G9_LDS u32x4 *>(s + WB + j * 8192 + at);
                rows_product<T>(w, x, sizeof(T) == 4 ? sum[t % SUMS][j] : acc[j]);
            }
        }
        if constexpr (sizeof(T) == 4)
#pragma unroll
            for (int j = 0; j < MT; j++) acc[j] += sum[0][j] + sum[SUMS - 1][j];
    };
    if (ng > 0) {
#pragma unroll
        for (int s = 0; s < NS - 1; s++) issue(s, s);
        int st = 0, free = NS - 1;
        for (int j = 0; j < ng; j++) {
            g9::wait_vm<(NS - 2) * LPS>();
            g9::wait_lgkm0();
            __syncthreads();
            issue(j + NS - 1, free);
            products(lds + st * SB);
            free = st;
            st = st + 1 == NS ? 0 : st + 1;
        }
        g9::wait_vm<0>();
    }
    __syncthreads();
    if (a.K % GK && slice == a.slices - 1) {   // the end of k, with zeros past it
        auto fill = [&](const T *m, long long ld, int rows, int r0, int count, G9_LDS unsigned char *to) {   // rows r0 .. of a matrix of `rows`
            for (int i = threadIdx.x; i < count * 32; i += 512) {
                const int r = i / 32, c = i % 32;
                union { u32x4 v; T e[V]; } u;
#pragma unroll
                for (int e = 0; e < V; e++) u.e[e] = whole * GK + c * V + e < a.K ? m[(long long)min(r0 + r, rows - 1) * ld + whole * GK + c * V + e] : T(0);
                *reinterpret_cast<G9_LDS u32x4 *>(to + r * 512 + ((c ^ (r & 15)) << 4)) = u.v;
            }
        };
        fill(a.W, a.ldw, a.N, n0, 64, lds);
        fill(a.X, a.ldx, a.M, 0, 16 * MT, lds + WB);
        __syncthreads();
        products(lds);
        __syncthreads();
    }
    G9_LDS f32x4 *other = (G9_LDS f32x4 *)lds;
    if (half)
#pragma unroll
        for (int j = 0; j < MT; j++) other[(cols * MT + j) * 64 + lane] = acc[j];
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int j = 0; j < MT; j++) {   // lane 16g + r has columns 4g .. 4g + 3 of row r
        const f32x4 sum = acc[j] + other[(cols * MT + j) * 64 + lane];
        if (a.slices > 1) a.parts[((((long long)slice * (gridDim.x / a.slices) + tile) * 4 + cols) * MT + j) * 64 + lane] = sum;
        else rows_store(a, tile, cols, j, lane, sum);
    }
}
// The slices' sums, in their order.
template <class T, int MT>
__global__ void __launch_bounds__(256) linear_rows_sum_kernel(RowsArgs<T> a, int tiles) {
    const long long plane = (long long)tiles * 4 * MT * 64, i = (long long)blockIdx.x * 256 + threadIdx.x;
    f32x4 sum = a.parts[i];
    for (int s = 1; s < a.slices; s++) sum += a.parts[i + s * plane];
    const long long w = i >> 6;
    rows_store(a, (int)(w / (4 * MT)), (int)(w / MT % 4), (int)(w % MT), threadIdx.x & 63, sum);
}

}  // namespace g9llm
