// Products of two MX4 matrices on the 4-bit matrix cores.
#pragma once
#include "mx4_gemm_kernel.h"

namespace g9llm {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ i32x8 fp4_operand(u32x4 v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }

// A workgroup of 2 × 2 waves makes 256 rows × 256 columns, each wave 128 × 128 (T = 8 row tiles), with v_mfma_scale_f32_32x32x64 (37 clocks in
// a loop of one wave a SIMD, where 16x16x128 takes 29 for half the products): lane l holds row l % 32 of two row tiles and block
// 2u + l / 32 of a stage's 128 k, u = 0, 1. 32 instructions a stage and wave leave the path from L2 about 1100 clocks, and
// it passes 57 to 64 bytes a clock and CU. So A, which two waves share in turn, goes through LDS, its tiles as they lie (16 KiB in,
// 32 KiB read), and W goes from L2 to registers (32 KiB). 4096 × 11008 × 4096: 98 to 101 µs, matrix cores 56 % busy.
// Four stages of A are on the ring: while stage s is multiplied, its fragments for s + 1 are read and s + 2 to s + 4 are on their
// way (s + 4 into the place of s, whose fragments every wave has by then). A fragment of W is loaded as soon as its registers are
// free, a stage or more ahead. The scales of 512 k (a word per lane and row tile) come with every fourth stage, A's through
// LDS on a ring of two, W's to registers. In whole groups each wait counts the copies and loads behind what it waits for: none of them is
// conditional (past the end the last ones are fetched again), and the next group takes what they bring. The stages after the last
// whole group count nothing.
template <class O>
__global__ void __launch_bounds__(256, 1) mx4_gemm_q_tile_kernel(Mx4View A, Mx4View W, O *__restrict__ C, long long ldc, int mtiles, int ntiles) {
    constexpr int T = 8, STAGE = 2 * T * 1024, NS = 4, SCALES = 2 * T * 256, T2 = T / 2, CP = T2, OPS = CP + T;   // copies of A, and all copies and loads, a stage and wave
    __shared__ __attribute__((aligned(16))) unsigned char smem[NS * STAGE + 2 * SCALES];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int total = mtiles * ntiles, run = (total + 7) / 8, id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= run || id >= total) return;
    // An XCD's run goes through bands of 8 row tiles, column by column: its 32 CUs then share 8 tiles of A and 4 of W.
    const int band = id / (8 * ntiles), high = min(mtiles - band * 8, 8), in_band = id - band * 8 * ntiles;
    const int mt0 = (band * 8 + in_band % high) * 2 * T, nt0 = in_band / high * 2 * T;   // first row tiles of A and of W
    const unsigned lds0 = (unsigned)(uintptr_t)(const G9_LDS unsigned char *)smem;
    // a wave copies row tiles wv·T/2 .. of a stage; a KiB of scales are those of four row tiles
    const uint8_t *src[CP], *ssrc;
#pragma unroll
    for (int j = 0; j < CP; j++) src[j] = A.codes + (long long)min(mt0 + wv * CP + j, A.rt - 1) * A.kc * 1024 + lane * 16;
    ssrc = A.scales + (long long)min(mt0 + wv * 4 + (lane >> 4), A.rt - 1) * A.kg * 256 + (lane & 15) * 16;
    auto dma = [](const void *p, unsigned lds) {
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(lds) : "memory");
    };
    auto issue_one = [&](int c, int j) {   // copy j of stage c
        dma(src[j] + (long long)min(c, A.kc - 1) * 1024, __builtin_amdgcn_readfirstlane(lds0 + (c & 3) * STAGE + (wv * CP + j) * 1024));
    };
    f32x16 acc[T2][T2];   // [32 columns][32 rows]
#pragma unroll
    for (int n = 0; n < T2; n++)
#pragma unroll
        for (int m = 0; m < T2; m++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[n][m][i] = 0.f;
    const int wm = (wv >> 1) * T, wn = (wv & 1) * T;   // the wave's first row tiles of the workgroup's
    const int half = lane >> 5, row32 = lane & 31;
    const int in_tile = 16 * half + (row32 & 15);   // 16-byte place of a fragment in its row tile (u adds 32), and word of its scale
    // W: a pair of row tiles from a uniform address, the lanes of its second tile further on (columns past the last repeat it)
    const uint8_t *wc[T2], *ws[T2];
    unsigned wo[T2], so[T2];
#pragma unroll
    for (int n = 0; n < T2; n++) {
        const int t0 = min(nt0 + wn + 2 * n, W.rt - 1), t1 = min(t0 + 1, W.rt - 1);
        wc[n] = W.codes + (long long)t0 * W.kc * 1024, ws[n] = W.scales + (long long)t0 * W.kg * 256;
        const unsigned up = row32 >= 16 ? t1 - t0 : 0;
        wo[n] = up * W.kc * 1024 + in_tile * 16, so[n] = up * W.kg * 256 + in_tile * 4;
    }
    const G9_LDS unsigned char *base = (const G9_LDS unsigned char *)smem;
    u32x4 a[2][T], w[2][T];   // fragments t = u·T/2 + 32-row tile of a stage, by its parity
    int sa[T], sw[T], sa_next[T], sw_next[T];
    // waits for a stage, behind which N copies and loads may be on their way, and for this wave's LDS reads, then for the other waves
    auto arrive = [](auto NN) {
        constexpr int N = decltype(NN)::value;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto load_one = [&](int c, auto JJ, int t) {   // fragment t of W of stage c, of parity JJ
        constexpr int j = decltype(JJ)::value;
        w[j][t] = *reinterpret_cast<const u32x4 *>(wc[t % T2] + ((long long)min(c, W.kc - 1) * 1024 + t / T2 * 512) + wo[t % T2]);
    };
    auto scales = [&](int c) {   // of the group that stage c begins
        const int grp = min(c / 4, A.kg - 1);
        dma(ssrc + grp * 256, __builtin_amdgcn_readfirstlane(lds0 + NS * STAGE + (c / 4 & 1) * SCALES + wv * 1024));
#pragma unroll
        for (int t = 0; t < T; t++) sw_next[t] = *reinterpret_cast<const int *>(ws[t % T2] + (grp * 256 + t / T2 * 128) + so[t % T2]);
    };
    auto read_scales = [&](int grp) {
        const G9_LDS int *s = (const G9_LDS int *)(base + NS * STAGE + (grp & 1) * SCALES) + wm * 64 + (row32 >> 4) * 64 + in_tile;
#pragma unroll
        for (int t = 0; t < T; t++) sa_next[t] = s[(t % T2) * 128 + t / T2 * 32];
    };
    auto read_one = [&](auto J, int t) {   // fragment t of A of a stage in place J of the ring
        constexpr int j = decltype(J)::value;
        a[j & 1][t] = ((const G9_LDS u32x4 *)(base + j * STAGE) + (wm + (row32 >> 4)) * 64 + in_tile)[(t % T2) * 128 + t / T2 * 32];
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    scales(0);
#pragma unroll
    for (int t = 0; t < T; t++) load_one(0, even, t);
#pragma unroll
    for (int t = 0; t < T2; t++) load_one(1, odd, t);
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int j = 0; j < CP; j++) issue_one(c, j);
    arrive(std::integral_constant<int, 3 * CP>());
#pragma unroll
    for (int t = 0; t < T; t++) read_one(even, t);
    read_scales(0);
    // A stage. With the matrix instructions of each fragment of A go a copy (in the first half), a fragment of the next stage, and
    // a load into the registers of W that the last half has left: the second half of the next stage, then the first of the one after.
    auto multiply = [&](int c0, auto J, auto COPY) __attribute__((always_inline)) {   // called seven times: what it refers to must stay in registers
        constexpr int j = decltype(J)::value;
        constexpr std::integral_constant<int, (j & 1)> here{};
        constexpr std::integral_constant<int, ((j + 1) & 1)> next{};
#pragma unroll
        for (int t = 0; t < T; t++) {
            if (decltype(COPY)::value && t < CP) issue_one(c0 + j + 4, t);
            read_one(std::integral_constant<int, (j + 1) % 4>(), t);
            if (j == 3 && t == T - 1) read_scales(c0 / 4 + 1);
            const int u = t / T2, m = t % T2;
#pragma unroll
            for (int n = 0; n < T2; n++)
                acc[n][m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(w[j & 1][u * T2 + n]), fp4_operand(a[j & 1][t]), acc[n][m], 4, 4, j,
                                                                            sw[u * T2 + n], j, sa[t]);
            if (t < T2) load_one(c0 + j + 1, next, T2 + t);
            else load_one(c0 + j + 2, here, t - T2);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto step = [&](int c0, auto J, bool first) __attribute__((always_inline)) {
        constexpr int j = decltype(J)::value;
        // what the two stages before this one have queued may be on its way, with the scales if one of them began a group; in
        // the first group the copies of stage 2 (and 3) stand for them
        if (first && j < 2) arrive(std::integral_constant<int, j == 0 ? 2 * CP : CP + OPS + 1 + T>());
        else arrive(std::integral_constant<int, 2 * OPS + (j == 1 || j == 2 ? 1 + T : 0)>());
        if (j == 0) scales(c0 + 4);
        multiply(c0, J, std::true_type());
    };
    auto take_scales = [&] {
#pragma unroll
        for (int t = 0; t < T; t++) sa[t] = sa_next[t], sw[t] = sw_next[t];
    };
    auto group = [&](int c0, bool first) __attribute__((always_inline)) {
        take_scales();
        step(c0, std::integral_constant<int, 0>(), first);
        step(c0, std::integral_constant<int, 1>(), first);
        step(c0, std::integral_constant<int, 2>(), first);
        step(c0, std::integral_constant<int, 3>(), first);
    };
    int c0 = 0;
    if (A.kc >= 4) {
        group(0, true);
        for (c0 = 4; c0 + 4 <= A.kc; c0 += 4) group(c0, false);
    }
    // The last one to three stages. Their copies are on their way, so nothing is queued but what they still take of W, and one wait
    // for all of it stands before them: a count would be wrong here, as the compiler drops loads that no stage uses.
    if (c0 < A.kc) {
        arrive(std::integral_constant<int, 0>());
        take_scales();
        multiply(c0, std::integral_constant<int, 0>(), std::false_type());
        if (c0 + 1 < A.kc) multiply(c0, std::integral_constant<int, 1>(), std::false_type());
        if (c0 + 2 < A.kc) multiply(c0, std::integral_constant<int, 2>(), std::false_type());
    }
    g9::wait_vm<0>();   // no copy may land after the workgroup has gone
    // lane l: row l % 32, and of register 4q + j column 8q + 4·(l / 32) + j. Both halves' 32-row tiles m go through LDS together.
    constexpr int COLS = 32 * T, PITCH = COLS * sizeof(O) + 16;
    static_assert(64 * PITCH <= sizeof(smem), "64 rows of the tile");
#pragma unroll
    for (int m = 0; m < T2; m++) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < T2; n++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                typedef O O4 __attribute__((ext_vector_type(4)));
                const f32x16 &v = acc[n][m];
                *reinterpret_cast<G9_LDS O4 *>((G9_LDS unsigned char *)smem + ((wv >> 1) * 32 + row32) * PITCH + (wn * 16 + n * 32 + 8 * q + 4 * half) * sizeof(O)) =
                    O4{(O)v[4 * q], (O)v[4 * q + 1], (O)v[4 * q + 2], (O)v[4 * q + 3]};
            }
        __syncthreads();
        store_rows<O, 256, 64, COLS, PITCH>((const G9_LDS unsigned char *)smem, W.rows - nt0 * 16, [&](int i) {
            const int row = (mt0 + i / 32 * T + 2 * m) * 16 + i % 32;
            return row < A.rows ? C + row * ldc + nt0 * 16 : (O *)nullptr;
        });
    }
}

// The same for fewer tiles: 128 rows × 128 columns a workgroup, two a CU, each wave 64 × 64. Its stage takes a quarter of the time, so
// both operands go through the ring of four stages, which gives a load three stages to arrive (1000 × 4096 × 4096 15.8 µs, the kernel above
// at T = 4 18.1). A stage is 128 k: 16 tiles of 1 KiB, A's, then W's; the scales of 512 k ride in front of every fourth stage.
template <class O>
__global__ void __launch_bounds__(256, 2) mx4_gemm_q_ring_kernel(Mx4View A, Mx4View W, O *__restrict__ C, long long ldc, int mtiles, int ntiles) {
    constexpr int T = 4, STAGE = 4 * T * 1024, NS = 4, SCALES = 4 * T * 256;
    constexpr int CP = T, SP = T / 4;   // copies per wave: of a stage's codes, and of a group's scales
    constexpr int RING_LDS = NS * STAGE + 2 * SCALES;
    __shared__ __attribute__((aligned(16))) unsigned char smem[RING_LDS];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int total = mtiles * ntiles, run = (total + 7) / 8, id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= run || id >= total) return;
    const int mt0 = id % mtiles * 2 * T, nt0 = id / mtiles * 2 * T;   // first row tiles of A and of W
    const unsigned lds0 = (unsigned)(uintptr_t)(const G9_LDS unsigned char *)smem;
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
    auto issue_scales = [&](int c) {   // in front of stage c, which begins a group
        const int grp = min(c / 4, A.kg - 1);
#pragma unroll
        for (int j = 0; j < SP; j++)
            dma(ssrc[j] + grp * 256, __builtin_amdgcn_readfirstlane(lds0 + NS * STAGE + (c / 4 & 1) * SCALES + (wv * SP + j) * 1024));
    };
    auto issue_one = [&](int c, int j) {   // copy j of stage c
        dma(src[j] + (long long)min(c, A.kc - 1) * 1024, __builtin_amdgcn_readfirstlane(lds0 + (c & 3) * STAGE + (wv * CP + j) * 1024));
    };
    constexpr int T2 = T / 2;
    f32x16 acc[T2][T2];   // [32 columns][32 rows]
#pragma unroll
    for (int n = 0; n < T2; n++)
#pragma unroll
        for (int m = 0; m < T2; m++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[n][m][i] = 0.f;
    const int wm = (wv >> 1) * T, wn = 2 * T + (wv & 1) * T;   // the wave's first tiles of a stage
    const G9_LDS unsigned char *base = (const G9_LDS unsigned char *)smem;
    const int half = lane >> 5, row32 = lane & 31;
    const int at = (row32 >> 4) * 64 + 16 * half + (row32 & 15);   // of a fragment: 16-byte place (u adds 32), and word of its scale
    u32x4 a[2][T], w[2][T];   // fragments t = u·T/2 + 32-row tile of a stage, by its parity
    int sa[T], sw[T], sa_next[T], sw_next[T];
    // waits for a stage, behind which N copies may be on their way, and for this wave's LDS reads, then for the other waves
    auto arrive = [](auto NN) {
        constexpr int N = decltype(NN)::value;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto read_scales = [&](int grp) {
        const G9_LDS int *s = (const G9_LDS int *)(base + NS * STAGE + (grp & 1) * SCALES) + at;
#pragma unroll
        for (int t = 0; t < T; t++) {
            const int o = (t % T2) * 128 + t / T2 * 32;
            sa_next[t] = s[wm * 64 + o], sw_next[t] = s[wn * 64 + o];
        }
    };
    auto read_one = [&](auto J, int t) {   // fragments t of a stage in place J of the ring
        constexpr int j = decltype(J)::value;
        const G9_LDS u32x4 *st = (const G9_LDS u32x4 *)(base + j * STAGE) + at + (t % T2) * 128 + t / T2 * 32;
        w[j & 1][t] = st[wn * 64], a[j & 1][t] = st[wm * 64];
    };
    issue_scales(0);
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int j = 0; j < CP; j++) issue_one(c, j);
    arrive(std::integral_constant<int, 3 * CP>());
#pragma unroll
    for (int t = 0; t < T; t++) read_one(std::integral_constant<int, 0>(), t);
    read_scales(0);
    // a stage: between the matrix instructions of a fragment of A, one copy and two of the next stage's fragments
    auto step = [&](int c0, auto J) {
        constexpr int j = decltype(J)::value;
        // stages + 2 and + 3 may be on their way, one of them with scales where it begins a group
        arrive(std::integral_constant<int, 2 * CP + (j == 1 || j == 2 ? SP : 0)>());
        if (j == 0) issue_scales(c0 + 4);
#pragma unroll
        for (int t = 0; t < T; t++) {
            issue_one(c0 + j + 4, t);
            read_one(std::integral_constant<int, (j + 1) % 4>(), t);
            if (j == 3 && t == T - 1) read_scales(c0 / 4 + 1);
            const int u = t / T2, m = t % T2;
#pragma unroll
            for (int n = 0; n < T2; n++)
                acc[n][m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(w[j & 1][u * T2 + n]), fp4_operand(a[j & 1][t]), acc[n][m], 4, 4, j,
                                                                            sw[u * T2 + n], j, sa[t]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int c0 = 0;
    for (; c0 + 4 <= A.kc; c0 += 4) {
#pragma unroll
        for (int t = 0; t < T; t++) sa[t] = sa_next[t], sw[t] = sw_next[t];
        step(c0, std::integral_constant<int, 0>());
        step(c0, std::integral_constant<int, 1>());
        step(c0, std::integral_constant<int, 2>());
        step(c0, std::integral_constant<int, 3>());
    }
    if (c0 < A.kc) {
#pragma unroll
        for (int t = 0; t < T; t++) sa[t] = sa_next[t], sw[t] = sw_next[t];
        step(c0, std::integral_constant<int, 0>());
        if (c0 + 1 < A.kc) step(c0, std::integral_constant<int, 1>());
        if (c0 + 2 < A.kc) step(c0, std::integral_constant<int, 2>());
    }
    g9::wait_vm<0>();   // no copy may land after the workgroup has gone
    // lane l: row l % 32, and of register 4q + j column 8q + 4·(l / 32) + j. Both halves' 32-row tiles m go through LDS together.
    constexpr int COLS = 32 * T, PITCH = COLS * sizeof(O) + 16;
    static_assert(64 * PITCH <= RING_LDS, "64 rows of the tile");
#pragma unroll
    for (int m = 0; m < T2; m++) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < T2; n++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                typedef O O4 __attribute__((ext_vector_type(4)));
                const f32x16 &v = acc[n][m];
                *reinterpret_cast<G9_LDS O4 *>((G9_LDS unsigned char *)smem + ((wv >> 1) * 32 + row32) * PITCH + ((wn - 2 * T) * 16 + n * 32 + 8 * q + 4 * half) * sizeof(O)) =
                    O4{(O)v[4 * q], (O)v[4 * q + 1], (O)v[4 * q + 2], (O)v[4 * q + 3]};
            }
        __syncthreads();
        store_rows<O, 256, 64, COLS, PITCH>((const G9_LDS unsigned char *)smem, W.rows - nt0 * 16, [&](int i) {
            const int row = (mt0 + i / 32 * T + 2 * m) * 16 + i % 32;
            return row < A.rows ? C + row * ldc + nt0 * 16 : (O *)nullptr;
        });
    }
}

}  // namespace g9llm
