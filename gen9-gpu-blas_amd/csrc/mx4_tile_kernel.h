// Products of many rows with MX4 weights: tiles of BM rows × 256 columns on the FP16 or BF16 matrix cores.
#pragma once
#include "mx4_gemm_kernel.h"

namespace g9llm {

// Activations as the tile kernel stages them: P planes of FP16 or BF16 rows, zeros up to a multiple of 128 k, 16-byte aligned.
struct Planes {
    const uint16_t *p;
    long long ld, plane;   // row stride and plane stride (elements)
};

// One 16-byte global→LDS copy per lane, lane L to lds + 16·L, from 64-bit addresses (see lds_dma16 for the waits).
__device__ __forceinline__ void lds_dma16_ptr(const void *p, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(lds) : "memory");
}

// A workgroup's 4 waves lie side by side in n: each makes all BM = 16·MT rows × 64 columns (4 column tiles; gated: 2 of W and
// 2 of the gate). Per 128 k and wave that is 16·MT matrix instructions to 64 conversions, and the weights, which no other
// wave needs, go from global memory to registers and are converted there. The rows are staged in LDS by direct copies, two
// stages: stage s + 1 is on its way while s is multiplied. 16-byte piece q of row m lies at q ^ (m & 15): eight lanes that
// read together then cover all banks.
template <class T, class O, int MT, bool GROUPED, bool GATED>
__global__ void __launch_bounds__(256, 2) mx4_gemm_tile_kernel(Planes A, Rows R, Mx4View W, Mx4View G, int experts, int mtiles, int ntiles) {
    typedef Act<T> X;
    typedef typename X::Frag Frag;
    constexpr int P = X::P, BM = MT * 16, NT = 4, PER = BM / 16;   // PER: copies per thread and stage
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * BM * 256];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    // Each XCD (workgroups b, b + 8, ...) takes a contiguous run of tiles, so that those resident on it share rows and weights.
    if (GROUPED) mtiles = R.tiles[-1];
    const int total = mtiles * ntiles, run = (total + 7) / 8, id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= run || id >= total) return;
    const int mt0 = GROUPED ? id / ntiles : id % mtiles, nt0 = GROUPED ? id % ntiles : id / mtiles;
    int first, count, e = 0;
    if (GROUPED) {
        e = R.tiles[2 * mt0], first = R.tiles[2 * mt0 + 1];
        count = min(BM, R.off[e + 1] - first);
    } else
        first = mt0 * BM, count = min(BM, R.M - first);
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
        const u32x4 *wc[NT];
        const unsigned *ws[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const Mx4View &V = GATED && n >= 2 ? G : W;
            const long long t = (long long)e * W.rt + min(tile[n], W.rt - 1);   // columns past the last repeat it and are not stored
            wc[n] = reinterpret_cast<const u32x4 *>(V.codes) + t * W.kc * 64 + lane;
            ws[n] = reinterpret_cast<const unsigned *>(V.scales) + t * W.kg * 64 + lane;
            top[n] = row_top(V.top + (t * 16 + r) * W.kt, W.kt);
        }
        // copy j of a thread: row (wv·PER + j)·4 + lane/16 of the tile, piece (lane & 15) ^ (row & 15); rows past the last repeat it
        const uint16_t *src[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int m = (wv * PER + j) * 4 + (lane >> 4), i = first + min(m, count - 1);
            long long row = i;
            if (GROUPED) row = R.lds ? R.order[i] : R.order[i] / R.S;
            src[j] = A.p + row * A.ld + ((lane & 15) ^ (m & 15)) * 8;
        }
        const unsigned lds0 = (unsigned)(uintptr_t)(const G9_LDS unsigned char *)smem + wv * PER * 1024;
        auto issue = [&](int stage, int buf) {   // stage = chunk·P + plane
            const long long at = (long long)(stage / P) * 128 + (stage % P) * A.plane;
#pragma unroll
            for (int j = 0; j < PER; j++) lds_dma16_ptr(src[j] + at, __builtin_amdgcn_readfirstlane(lds0 + buf * BM * 256 + j * 1024));
        };
        u32x4 w[NT], wn[NT];
        unsigned sw[NT], sn[NT];
        issue(0, 0);
#pragma unroll
        for (int n = 0; n < NT; n++) wn[n] = wc[n][0], sn[n] = ws[n][0];
        const int stages = W.kc * P;
        float sc[NT];
        for (int s = 0; s < stages; s++) {
            const int c = s / P;
            g9::wait_vm<0>();
            __syncthreads();
            if (P == 1 || s % P == 0) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    w[n] = wn[n];
                    if (c % 4 == 0) sw[n] = sn[n];
                    sc[n] = X::scale(sw[n] >> (c % 4 * 8) & 255u, top[n]);
                }
            }
            if (s + 1 < stages) {
                issue(s + 1, (s + 1) & 1);
                if ((P == 1 || s % P == 0) && c + 1 < W.kc) {
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        wn[n] = wc[n][(c + 1) * 64];
                        if (c % 4 == 3) sn[n] = ws[n][(c + 1) / 4 * 64];
                    }
                }
            }
            const G9_LDS unsigned char *base = (const G9_LDS unsigned char *)smem + (s & 1) * BM * 256 + r * 256;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                Frag a[MT], b[NT];
#pragma unroll
                for (int m = 0; m < MT; m++) a[m] = *reinterpret_cast<const G9_LDS Frag *>(base + m * 4096 + (((4 * g + i) ^ r) << 4));
#pragma unroll
                for (int n = 0; n < NT; n++) b[n] = X::weights(w[n][i], sc[n]);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int n = 0; n < NT; n++) acc[n][m] = X::mfma(b[n], a[m], acc[n][m]);
            }
        }
    }
    int tn[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) tn[n][j] = __shfl(top[n], 4 * g + j);
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int i = m * 16 + r;
        if (i >= count) continue;
        O *c;
        if (GROUPED) {
            const int slot = R.order[first + i];
            c = (O *)R.C + (slot / R.S) * R.ldct + (slot % R.S) * R.ldcs;
        } else
            c = (O *)R.C + (long long)(first + i) * R.ldct;
#pragma unroll
        for (int n = 0; n < (GATED ? 2 : NT); n++) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                y[j] = X::finish(acc[n][m][j], tn[n][j]);
                if (GATED) y[j] *= silu(X::finish(acc[(n + 2) % NT][m][j], tn[(n + 2) % NT][j]));
            }
            const int col = tile[n] * 16 + 4 * g;
            if (col + 4 <= W.rows) {
                typedef O O4 __attribute__((ext_vector_type(4), aligned(sizeof(O))));
                *reinterpret_cast<O4 *>(c + col) = O4{(O)y[0], (O)y[1], (O)y[2], (O)y[3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (col + j < W.rows) c[col + j] = (O)y[j];
            }
        }
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
