// Products of many rows with MX4 weights: tiles of 64 rows × 256 columns on the FP16 or BF16 matrix cores.
#pragma once
#include "mx4_rows_kernel.h"

namespace g9llm {

// Activations as the tile kernel stages them: P planes of FP16 or BF16 rows, zeros up to a multiple of 128 k, 16-byte aligned.
struct Planes {
    const uint16_t *p;
    long long ld, plane;   // row stride and plane stride (elements)
};

// 64 rows × 256 columns a workgroup, 4 waves side by side in n: each all rows × 64 columns (4 column tiles; gated: 2 of W and 2
// of the gate), three workgroups a CU. Per 128 k and wave that is 64 matrix instructions to 64 conversions, which run beside
// them, and the weights, which no other wave needs, go from global memory to registers and are converted there. The rows are
// staged in LDS by direct copies, two stages: stage s + 1 is on its way while s is multiplied. Their fragments are read three
// ahead of the one that is multiplied: at their full rate the matrix cores take 64 bytes a clock and CU, about half of what ds_read_b128 gives.
// FP16 1000 × 11008 × 4096: 80 µs, 1.13 PFLOP/s, near what a large FP16 product reaches on this GPU (1.1 to 1.3); with no loads from memory at
// all the loop takes 59 µs. Tiles of 128 rows, of 512 columns, and one wave a SIMD with 64 × 512 were not faster.
template <class T, class O, bool GROUPED, bool GATED>
__global__ void __launch_bounds__(256, 3) mx4_gemm_tile_kernel(Planes A, Rows R, Mx4View W, Mx4View G, int experts, int mtiles, int ntiles) {
    typedef Act<T> X;
    typedef typename X::Frag Frag;
    constexpr int P = X::P, MT = 4, NT = 4, STAGE = MT * 4096;
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * STAGE + 1024];   // two stages, or a finished tile of FP16 with its rows 16 bytes apart
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    // Each XCD (workgroups b, b + 8, ...) takes a contiguous run of tiles, so that those resident on it share rows and weights.
    if (GROUPED) mtiles = R.tiles[-1];
    const int total = mtiles * ntiles, run = (total + 7) / 8, id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= run || id >= total) return;
    const int mt0 = GROUPED ? id / ntiles : id % mtiles, nt0 = GROUPED ? id % ntiles : id / mtiles;
    int first, count, e = 0;
    if (GROUPED) {
        e = R.tiles[2 * mt0], first = R.tiles[2 * mt0 + 1];
        count = min(MT * 16, R.off[e + 1] - first);
    } else
        first = mt0 * MT * 16, count = min(MT * 16, R.M - first);
    int tile[NT];   // row tiles of W (gated: 2 of W, the same 2 of G)
#pragma unroll
    for (int n = 0; n < NT; n++) tile[n] = GATED ? (nt0 * 4 + wv) * 2 + n % 2 : (nt0 * 4 + wv) * 4 + n;

    f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int m = 0; m < MT; m++) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    int top[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) top[n] = 0;

    if (!GROUPED || e < experts) {
        const uint8_t *wc[NT], *ws[NT], *tops[NT];   // uniform: the lane is added to each load's offset
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const Mx4View &V = GATED && n >= 2 ? G : W;
            const long long t = (long long)e * W.rt + min(tile[n], W.rt - 1);   // columns past the last repeat it and are not stored
            wc[n] = V.codes + t * W.kc * 1024;
            ws[n] = V.scales + t * W.kg * 256;
            tops[n] = V.top + (t * 16 + r) * W.kt;
        }
        if (P == 1) row_tops<NT>(tops, W.kt, top);
        // copy j of a thread: row (wv·MT + j)·4 + lane/16 of the tile, piece (lane & 15) ^ swizzle(row); rows past the last repeat it
        const uint16_t *src[MT];
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int m = (wv * MT + j) * 4 + g, i = first + min(m, count - 1);
            long long row = i;
            if (GROUPED) row = R.lds ? R.order[i] : R.order[i] / R.S;
            src[j] = A.p + row * A.ld + (r ^ swizzle(m)) * 8;
        }
        const unsigned lds0 = (unsigned)(uintptr_t)(const G9_LDS unsigned char *)smem + wv * MT * 1024;
        auto issue = [&](int s) {   // the rows of stage s = chunk · P + plane
            const long long at = (long long)(s / P) * 128 + s % P * A.plane;
#pragma unroll
            for (int j = 0; j < MT; j++)
                asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                             : : "v"(src[j] + at), "s"(__builtin_amdgcn_readfirstlane(lds0 + (s & 1) * STAGE + j * 1024)) : "memory");
        };
        u32x4 w[NT], wn[NT];
        unsigned sn[NT];
        float sc[NT];
        auto fetch = [&](int c) {
            // the lane's offset made anew: as a loop invariant it would be added to each address beforehand, in 16 registers too many
            unsigned at = lane * 16;
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int n = 0; n < NT; n++) {
                wn[n] = *reinterpret_cast<const u32x4 *>(wc[n] + (long long)c * 1024 + at);
                sn[n] = (ws[n] + (c / 4 * 256 + c % 4))[at / 4];
            }
        };
        const int stages = W.kc * P, sw_r = swizzle(r);
        const G9_LDS unsigned char *base = (const G9_LDS unsigned char *)smem + r * 256;
        int q[4];   // where this lane's pieces of a step lie in its row
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = ((4 * g + i) ^ sw_r) << 4;
        issue(0);
        fetch(0);
        for (int s = 0; s < stages; s++) {
            const int c = s / P;
            g9::wait_vm<0>();
            __syncthreads();
            if (P == 1 || s % P == 0) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    w[n] = wn[n];
                    sc[n] = X::scale(sn[n], top[n]);
                }
            }
            if (s + 1 < stages) {
                issue(s + 1);
                if (P == 1 || s % P == 0) fetch(min(c + 1, W.kc - 1));
            }
            const G9_LDS unsigned char *st = base + (s & 1) * STAGE;
            Frag a[4], b[NT];
            auto read = [&](int t) { a[t & 3] = *reinterpret_cast<const G9_LDS Frag *>(st + t % MT * 4096 + q[t / MT]); };
            read(0);
            read(1);
            read(2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < 4 * MT; t++) {
                if (t + 3 < 4 * MT) read(t + 3);
                if (t % MT == 0)
#pragma unroll
                    for (int n = 0; n < NT; n++) b[n] = X::weights(w[n][t / MT], sc[n]);
#pragma unroll
                for (int n = 0; n < NT; n++) acc[n][t % MT] = X::mfma(b[n], a[t & 3], acc[n][t % MT]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    constexpr int NO = GATED ? NT / 2 : NT, COLS = NO * 64;   // column tiles a wave, columns a workgroup
    int ty[NO][4], tz[NO][4];
#pragma unroll
    for (int n = 0; n < NO; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) ty[n][j] = __shfl(top[n], 4 * g + j), tz[n][j] = GATED ? __shfl(top[(n + 2) % NT], 4 * g + j) : 0;
    // the tile through LDS in one piece (FP16) or two (FP32)
    typedef O O4 __attribute__((ext_vector_type(4)));
    constexpr int PIECE = sizeof(O) == 2 ? 64 : 32, PITCH = COLS * sizeof(O) + 16;
    static_assert(PIECE * PITCH <= sizeof(smem), "a piece of the tile");
#pragma unroll
    for (int p = 0; p < 64; p += PIECE) {
        __syncthreads();
#pragma unroll
        for (int m = p / 16; m < (p + PIECE) / 16; m++)
#pragma unroll
            for (int n = 0; n < NO; n++) {
                O4 v;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float y = X::finish(acc[n][m][j], ty[n][j]);
                    if (GATED) y *= silu(X::finish(acc[(n + 2) % NT][m][j], tz[n][j]));
                    v[j] = (O)y;
                }
                *reinterpret_cast<G9_LDS O4 *>((G9_LDS unsigned char *)smem + (m * 16 + r - p) * PITCH + ((wv * NO + n) * 16 + 4 * g) * sizeof(O)) = v;
            }
        __syncthreads();
        store_rows<O, 256, PIECE, COLS, PITCH>((const G9_LDS unsigned char *)smem, W.rows - nt0 * COLS, [&](int i) {
            if (p + i >= count) return (O *)nullptr;
            long long at;
            if (GROUPED) {
                const int slot = R.order[first + p + i];
                at = slot / R.S * R.ldct + slot % R.S * R.ldcs;
            } else
                at = (long long)(first + p + i) * R.ldct;
            return (O *)R.C + at + nt0 * COLS;
        });
    }
}

// Rows of activations to planes: T·S rows at X + t·ldt + s·lds, each thread eight k.
template <class T>
__global__ void __launch_bounds__(256) mx4_planes_kernel(const T *__restrict__ X, long long ldt, long long lds, int S, long long rows, int K, int octets,
                                                         uint16_t *__restrict__ out, long long plane) {
    typedef Act<T> A;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * octets) return;
    const long long row = i / octets;
    const int k = (int)(i % octets) * 8;
    T v[8];
    load8(X + row / S * ldt + row % S * lds, k, K, v);
    typename A::Frag f[A::P];
    A::split(v, f);
#pragma unroll
    for (int p = 0; p < A::P; p++) *reinterpret_cast<typename A::Frag *>(out + p * plane + row * octets * 8 + k) = f[p];
}

// FP16 rows that lie in whole 128-k chunks at 4-byte alignment are taken in place; others, and FP32 ones, go through the
// work space (their rows T·S, or T where the places of a token share a row: lds = 0).
template <class T> int stage_planes(const Rows &R, int T_, int K, int kc, Planes *out) {
    const long long S = R.lds ? R.S : 1, rows = T_ * S;
    if (sizeof(T) == 2 && K % 128 == 0 && ((uintptr_t)R.A & 3) == 0 && R.ldt % 2 == 0 && (S == 1 || R.ldt == S * R.lds) && R.lds % 2 == 0) {
        *out = {(const uint16_t *)R.A, S == 1 ? R.ldt : R.lds, 0};
        return 0;
    }
    const int octets = kc * 16;
    const long long plane = rows * octets * 8;
    if (cdiv(rows * octets, 256) > 0xffffff) G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "more rows than one launch can index");
    void *p = nullptr;
    G9_TRY(scratch(SLOT_A, (size_t)plane * Act<T>::P * 2, &p));
    hipLaunchKernelGGL((mx4_planes_kernel<T>), dim3((unsigned)cdiv(rows * octets, 256)), dim3(256), 0, stream, (const T *)R.A, R.ldt, R.lds, (int)S, rows, K,
                       octets, (uint16_t *)p, plane);
    G9_HIP(hipGetLastError());
    *out = {(const uint16_t *)p, (long long)octets * 8, plane};
    return 0;
}

}  // namespace g9llm
