// Products of two MX4 matrices on the 4-bit matrix cores.
#pragma once
#include "llm.h"
#include "lds_dma.h"
#include <type_traits>

namespace g9llm {

typedef int i32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8 fp4_operand(u32x4 v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }

// A workgroup of 2 × 2 waves makes 32·T rows × 32·T columns, each wave 16·T × 16·T. A stage is 128 k: 4·T tiles of 1 KiB that
// go to LDS as they lie, so that every fragment is one conflict-free 16-byte read per lane. Four stages are on the ring: while
// stage s is multiplied, s + 1 to s + 3 are on their way. The scales of 512 k (a word per lane and row tile) ride in front of
// every fourth stage, on a ring of two. Copies past the last tile of k repeat it and are not multiplied, so that each
// wait knows how many copies follow what it waits for.
template <class O, int T>
__global__ void __launch_bounds__(256, T == 8 ? 1 : 2) mx4_gemm_q_tile_kernel(Mx4View A, Mx4View W, O *__restrict__ C, long long ldc, int mtiles, int ntiles) {
    constexpr int STAGE = 4 * T * 1024, NS = 4, SCALES = 4 * T * 256;
    constexpr int CP = T, SP = T / 4;   // copies per wave: of a stage's codes, and of a group's scales
    extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int total = mtiles * ntiles, run = (total + 7) / 8, id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= run || id >= total) return;
    const int mt0 = id % mtiles * 2 * T, nt0 = id / mtiles * 2 * T;   // first row tiles of A and of W
    const unsigned lds0 = (unsigned)(uintptr_t)(const G9_LDS unsigned char *)dyn;
    // tile t of a stage: row tile mt0 + t of A for t < 2T, nt0 + t − 2T of W after; a wave copies tiles wv·T .. wv·T + T − 1
    const uint8_t *src[CP], *ssrc[SP];
    auto rowtile = [&](int t) {
        return t < 2 * T ? min(mt0 + t, A.rt - 1) : min(nt0 + t - 2 * T, W.rt - 1);
    };
#pragma unroll
    for (int j = 0; j < CP; j++) {
        const int t = wv * CP + j;
        src[j] = (t < 2 * T ? A.codes : W.codes) + (long long)rowtile(t) * A.kc * 1024 + lane * 16;
    }
#pragma unroll
    for (int j = 0; j < SP; j++) {
        const int t = (wv * SP + j) * 4 + g;
        ssrc[j] = (t < 2 * T ? A.scales : W.scales) + (long long)rowtile(t) * A.kg * 256 + r * 16;
    }
    auto dma = [](const void *p, unsigned lds) {
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(lds) : "memory");
    };
    auto issue = [&](int c) {
        const int at = min(c, A.kc - 1);
        if (c % 4 == 0) {
            const int grp = min(c / 4, A.kg - 1);
#pragma unroll
            for (int j = 0; j < SP; j++)
                dma(ssrc[j] + grp * 256, __builtin_amdgcn_readfirstlane(lds0 + NS * STAGE + (c / 4 & 1) * SCALES + (wv * SP + j) * 1024));
        }
#pragma unroll
        for (int j = 0; j < CP; j++)
            dma(src[j] + (long long)at * 1024, __builtin_amdgcn_readfirstlane(lds0 + (c & 3) * STAGE + (wv * CP + j) * 1024));
    };
    f32x4 acc[T][T];   // [column tile][row tile]
#pragma unroll
    for (int n = 0; n < T; n++)
#pragma unroll
        for (int m = 0; m < T; m++) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    issue(0);
    issue(1);
    issue(2);
    const int wm = (wv >> 1) * T, wn = 2 * T + (wv & 1) * T;   // the wave's first tiles of a stage
    const G9_LDS unsigned char *base = (const G9_LDS unsigned char *)dyn;
    int sa[T], sw[T];
    for (int c0 = 0; c0 < A.kc; c0 += 4) {
        auto step = [&](auto J) {
            constexpr int j = decltype(J)::value;
            // stages c + 1 and c + 2 may be on their way, one of them with scales where it begins a group
            // (and no LDS read of this wave: the next copies go to the stage that it has just read)
            constexpr int N = 2 * CP + (j >= 2 ? SP : 0);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            issue(c0 + j + 3);
            if (j == 0) {
                const G9_LDS int *s = (const G9_LDS int *)(base + NS * STAGE + (c0 / 4 & 1) * SCALES) + lane;
#pragma unroll
                for (int t = 0; t < T; t++) sa[t] = s[(wm + t) * 64], sw[t] = s[(wn + t) * 64];
            }
            if (c0 + j < A.kc) {
                const G9_LDS u32x4 *st = (const G9_LDS u32x4 *)(base + j * STAGE) + lane;
                u32x4 a[T], w[T];
#pragma unroll
                for (int t = 0; t < T; t++) w[t] = st[(wn + t) * 64];
#pragma unroll
                for (int t = 0; t < T; t++) a[t] = st[(wm + t) * 64];
#pragma unroll
                for (int m = 0; m < T; m++)
#pragma unroll
                    for (int n = 0; n < T; n++)
                        acc[n][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(w[n]), fp4_operand(a[m]), acc[n][m], 4, 4, j, sw[n], j, sa[m]);
            }
        };
        step(std::integral_constant<int, 0>());
        step(std::integral_constant<int, 1>());
        step(std::integral_constant<int, 2>());
        step(std::integral_constant<int, 3>());
    }
    g9::wait_vm<0>();   // no copy may land after the workgroup has gone
#pragma unroll
    for (int m = 0; m < T; m++) {
        const int row = (mt0 + wm + m) * 16 + r;
        if (row >= A.rows) continue;
#pragma unroll
        for (int n = 0; n < T; n++) {
            const int col = (nt0 + wn - 2 * T + n) * 16 + 4 * g;
            O *c = C + row * ldc + col;
            if (col + 4 <= W.rows) {
                typedef O O4 __attribute__((ext_vector_type(4), aligned(sizeof(O))));
                *reinterpret_cast<O4 *>(c) = O4{(O)acc[n][m][0], (O)acc[n][m][1], (O)acc[n][m][2], (O)acc[n][m][3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (col + j < W.rows) c[j] = (O)acc[n][m][j];
            }
        }
    }
}

}  // namespace g9llm
