// Products of few rows with MX4 weights (decode): the weights are read once, straight into the registers that multiply them.
#pragma once
#include "mx4_gemm_kernel.h"

namespace g9llm {

// The rows of a tile, to `slots` in LDS: of the plan's tile t, or (ids: at most FEW_PLACES places, no plan) of place t's expert, if t is
// the first, 17th (ROWS + 1st), ... place with that expert; count 0 otherwise. e = experts: places without one. All threads of a
// workgroup call it.
constexpr int FEW_PLACES = 64;   // a place a lane
struct TileRows {
    int e, first, count;
};
template <int ROWS> __device__ __forceinline__ TileRows tile_rows(const Rows &R, int t, int experts, int *slots) {
    TileRows o;
    if (!R.ids) {
        o.e = R.tiles[2 * t], o.first = R.tiles[2 * t + 1];
        o.count = min(ROWS, R.off[o.e + 1] - o.first);
        if ((int)threadIdx.x < o.count) slots[threadIdx.x] = R.order[o.first + threadIdx.x];
    } else {
        const int lane = threadIdx.x & 63;
        const int expert = lane < R.M ? (int)min((unsigned)R.ids[lane], (unsigned)experts) : -1;   // ids outside 0..E−1: E
        o.e = __builtin_amdgcn_readlane(expert, t), o.first = 0;
        const unsigned long long mask = __ballot(expert == o.e);
        const int before = __builtin_popcountll(mask & ((1ull << t) - 1));
        o.count = before % ROWS ? 0 : min(ROWS, __builtin_popcountll(mask) - before);
        const int at = __builtin_popcountll(mask & ((1ull << lane) - 1)) - before;
        if (threadIdx.x < 64 && expert == o.e && at >= 0 && at < o.count) slots[at] = lane;
    }
    __syncthreads();
    return o;
}

// 32 consecutive k of a row in MFMA fragments: f[i][p] the i-th eight, piece p.
template <class T> struct Row32;
template <> struct Row32<_Float16> {
    u32x4 v[4];
    __device__ __forceinline__ void load(const _Float16 *p) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __builtin_bit_cast(u32x4, g9::load16u(p + 8 * i));
    }
    __device__ __forceinline__ void load_tail(const _Float16 *row, int k, int K) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            _Float16 e[8];
            load8(row, k + 8 * i, K, e);
            __builtin_memcpy(&v[i], e, 16);
        }
    }
    __device__ __forceinline__ void fragments(f16x8 (*f)[1]) const {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i][0] = __builtin_bit_cast(f16x8, v[i]);
    }
};
template <> struct Row32<float> {
    u32x4 v[8];
    __device__ __forceinline__ void load(const float *p) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __builtin_bit_cast(u32x4, g9::load16u(p + 4 * i));
    }
    __device__ __forceinline__ void load_tail(const float *row, int k, int K) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float e[8];
            load8(row, k + 8 * i, K, e);
            __builtin_memcpy(&v[2 * i], e, 32);
        }
    }
    // Act<float>::split without its test of each element: an infinity or NaN leaves a NaN in the last piece, and only then
    // are the elements split again with the test.
    __device__ __forceinline__ void fragments(bf16x8 (*f)[3]) const {
        float any = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            u32x4 q[3];
#pragma unroll
            for (int h = 0; h < 4; h++) {
                unsigned p[3][2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const unsigned u = v[2 * i + h / 2][h % 2 * 2 + j];
                    p[0][j] = u & 0xffff0000u;
                    const float r = __builtin_bit_cast(float, u) - __builtin_bit_cast(float, p[0][j]);
                    p[1][j] = __builtin_bit_cast(unsigned, r) & 0xffff0000u;
                    const float l = r - __builtin_bit_cast(float, p[1][j]);
                    p[2][j] = __builtin_bit_cast(unsigned, l);
                    any += l;
                }
#pragma unroll
                for (int w = 0; w < 3; w++) q[w][h] = __builtin_amdgcn_perm(p[w][1], p[w][0], 0x07060302u);   // the high halves
            }
#pragma unroll
            for (int w = 0; w < 3; w++) f[i][w] = __builtin_bit_cast(bf16x8, q[w]);
        }
        if (__ballot(any != any)) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float e[8];
                __builtin_memcpy(e, &v[2 * i], 32);
                Act<float>::split(e, f[i]);
            }
        }
    }
};

// The end of a row's four columns col .. col + 3 (y: the sum with W, z: with the gate): to C, or (dense) as a part's sums.
template <class T, class O, bool GROUPED, bool GATED>
__device__ __forceinline__ void finish4(const Rows &R, const Mx4View &W, const Split &split, int part, int first, const int *slots, int i, int col, f32x4 y, f32x4 z,
                                        const int *ty, const int *tz) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        y[j] = Act<T>::finish(y[j], ty[j]);
        if (GATED) z[j] = Act<T>::finish(z[j], tz[j]);
    }
    if (!GROUPED && split.parts > 1) {
        if (col >= W.rows) return;   // ld is whole column tiles
        *reinterpret_cast<f32x4 *>(split.sums + ((long long)part * split.rows + first + i) * split.ld + col) = y;
        return;
    }
    O *c;
    if (GROUPED) {
        const int slot = slots[i];
        c = (O *)R.C + slot / R.S * R.ldct + slot % R.S * R.ldcs;
    } else
        c = (O *)R.C + (long long)(first + i) * R.ldct;
    if (GATED)
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] *= silu(z[j]);
    if (col + 4 <= W.rows) {
        typedef O O4 __attribute__((ext_vector_type(4), aligned(sizeof(O))));
        *reinterpret_cast<O4 *>(c + col) = O4{(O)y[0], (O)y[1], (O)y[2], (O)y[3]};
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (col + j < W.rows) c[col + j] = (O)y[j];
    }
}

// C from the parts' sums, the parts in their order: a thread for each element, so that few rows still fill the GPU, sixteen
// loads on their way at a time.
template <class O>
__global__ void __launch_bounds__(256) mx4_sum_parts_kernel(Rows R, Split split, int N) {
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x, row = at / split.ld;
    const int col = (int)(at % split.ld);
    if (row >= split.rows || col >= N) return;
    const float *p = split.sums + at;
    const long long plane = split.rows * split.ld;
    float y = 0.f;
    int k = 0;
    for (; k + 16 <= split.parts; k += 16) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = p[(k + i) * plane];
#pragma unroll
        for (int i = 0; i < 16; i++) y += v[i];
    }
    if (k < split.parts) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = k + i < split.parts ? p[(k + i) * plane] : 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) y += v[i];
    }
    ((O *)R.C)[row * R.ldct + col] = (O)y;
}

// A workgroup makes 16 rows of 16 columns (gated: of W and of the gate) by 4 waves along k; `split` workgroups share the k of
// a tile. Weights and rows of the next D chunks of 128 k are on their way in registers. Lane 16g + r multiplies columns' row r of
// each weight tile, activations' row r. FP16 1 × 11008 × 4096: 7.3 µs for 24 MB, about 3 of them what an empty kernel takes.
template <class T, class O, int D, bool GROUPED, bool GATED>
__global__ void __launch_bounds__(256) mx4_gemm_rows_kernel(Rows R, Mx4View W, Mx4View G, int experts, Split split) {
    typedef Act<T> X;
    typedef typename X::Frag Frag;
    constexpr int NW = GATED ? 2 : 1, WAVES = 4;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int part = blockIdx.x % split.parts, tile = blockIdx.x / split.parts;
    const int mt = tile / W.rt, nt = tile % W.rt;
    __shared__ int slots[GROUPED ? 16 : 1];
    int first = 0, count = min(16, R.M), e = 0;   // dense: one tile of rows
    if (GROUPED) {
        if (!R.ids && mt >= R.tiles[-1]) return;
        const TileRows o = tile_rows<16>(R, mt, experts, slots);
        e = o.e, first = o.first, count = o.count;
        if (count == 0) return;
    }
    f32x4 acc[NW];
    int top[NW];
#pragma unroll
    for (int q = 0; q < NW; q++) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f}, top[q] = 0;
    if (!GROUPED || e < experts) {
        const int i = min(r, count - 1);   // rows past the last repeat it and are not stored
        long long at;
        if (GROUPED) {
            const int slot = slots[i];
            at = slot / R.S * R.ldt + slot % R.S * R.lds;
        } else
            at = i * R.ldt;
        const T *row = (const T *)R.A + at + g * 32;
        const u32x4 *wc[NW];
        const uint8_t *ws[NW], *tops[NW];
#pragma unroll
        for (int q = 0; q < NW; q++) {
            const Mx4View &V = q ? G : W;
            const long long t = (long long)e * W.rt + nt;
            wc[q] = reinterpret_cast<const u32x4 *>(V.codes) + t * W.kc * 64 + lane;
            ws[q] = V.scales + t * W.kg * 256 + lane * 4;
            tops[q] = V.top + (t * 16 + r) * W.kt;
        }
        if (X::P == 1) row_tops<NW>(tops, W.kt, top);
        const int ways = split.parts * WAVES, way = part * WAVES + wv, whole = W.K / 128;
        const int c1 = (int)((long long)whole * way / ways), end = (int)((long long)whole * (way + 1) / ways);
        u32x4 w[D][NW];
        unsigned s[D][NW];
        Row32<T> a[D];
        auto fetch_weights = [&](int c, int d) {
#pragma unroll
            for (int q = 0; q < NW; q++) {
                w[d][q] = __builtin_nontemporal_load(wc[q] + (long long)c * 64);
                s[d][q] = ws[q][c / 4 * 256 + c % 4];
            }
        };
        auto fetch = [&](int c, int d) {   // chunk c to the registers of place d
            fetch_weights(c, d);
            a[d].load(row + c * 128);
        };
        auto multiply = [&](int d) {
            Frag f[4][X::P];
            a[d].fragments(f);
#pragma unroll
            for (int q = 0; q < NW; q++) {
                const float sc = X::scale(s[d][q], top[q]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const Frag b = X::weights(w[d][q][i], sc);
#pragma unroll
                    for (int p = 0; p < X::P; p++) acc[q] = X::mfma(b, f[i][p], acc[q]);
                }
            }
        };
        if (c1 < end) {
            // No load is conditional (past the end the last chunk is loaded again): a wait then leaves all younger loads on their way.
#pragma unroll
            for (int d = 0; d < D; d++) fetch(min(c1 + d, end - 1), d);
            int c = c1;
            for (; c + D < end; c += D) {
#pragma unroll
                for (int d = 0; d < D; d++) {
                    multiply(d);
                    fetch(min(c + d + D, end - 1), d);
                }
            }
#pragma unroll
            for (int d = 0; d < D; d++)
                if (c + d < end) multiply(d);
        }
        if (W.K % 128 && way == ways - 1) {   // the chunk in which the rows end
            fetch_weights(whole, 0);
            a[0].load_tail(row - g * 32, whole * 128 + g * 32, W.K);
            multiply(0);
        }
    }
    // the sums of the waves along k, in their order
    __shared__ f32x4 sums[(WAVES - 1) * NW * 64];
    if (wv) {
#pragma unroll
        for (int q = 0; q < NW; q++) sums[((wv - 1) * NW + q) * 64 + lane] = acc[q];
    }
    __syncthreads();
    if (wv) return;
#pragma unroll
    for (int k = 1; k < WAVES; k++)
#pragma unroll
        for (int q = 0; q < NW; q++) acc[q] += sums[((k - 1) * NW + q) * 64 + lane];
    int tn[NW][4];
#pragma unroll
    for (int q = 0; q < NW; q++)
#pragma unroll
        for (int j = 0; j < 4; j++) tn[q][j] = __shfl(top[q], 4 * g + j);
    if (r < count) finish4<T, O, GROUPED, GATED>(R, W, split, part, first, slots, r, nt * 16 + 4 * g, acc[0], acc[NW - 1], tn[0], tn[NW - 1]);
}

// A barrier for what waves pass each other in LDS: their loads from memory stay on their way (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    g9::wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// 8 waves side by side in n, each 16·NT columns (gated: of W and of the gate) of MT·16 rows. The rows of each 128 k are taken
// apart once for the whole workgroup, into FP16 or BF16 planes in LDS (two buffers). A thread loads U elements at a time. Weights and rows of the next D
// chunks are on their way in registers; both, as loads return in order and the wait for the nearest rows would be a wait for
// all older weights too. FP32 24 × 4096 × 11008 in 8 parts of k: 15 to 16.5 µs for 24 MB of weights, 11 chunks of
// 1.4 µs. Of these the matrix cores are busy 0.3; each wave reads all rows in three planes for its 16 columns, 192 KiB a chunk, 0.6 µs at
// the 320 bytes a ns that eight waves read at if they do nothing else; the rest is the chain of split, barrier and first reads. 4 waves of 64 columns, two workgroups a CU, which read LDS half as often, took 18 to 20.
template <class T, class O, int MT, int NT, int D, bool GROUPED, bool GATED>
__global__ void __launch_bounds__(512, 2) mx4_gemm_few_kernel(Rows R, Mx4View W, Mx4View G, int experts, int mtiles, int ntiles, Split split) {
    typedef Act<T> X;
    typedef typename X::Frag Frag;
    constexpr int NW = GATED ? 2 : 1, P = X::P, PLANE = MT * 4096, NV = 8, NTH = NV * 64;
    constexpr int U = MT * 2048 / NTH < (int)(16 / sizeof(T)) ? MT * 2048 / NTH : 16 / sizeof(T);   // elements a load
    constexpr int PR = 128 / U, NL = MT * 16 * PR / NTH;                                            // threads a row, loads a thread
    typedef T TU __attribute__((ext_vector_type(U), aligned(sizeof(T))));
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * P * PLANE];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    // Each XCD (workgroups b, b + 8, ...) takes a contiguous run of tiles, so that those resident on it share rows and weights:
    // dense, row tiles of the same columns; experts, column tiles of the same rows.
    // Without a plan the places that come first have most of the work, so they are dealt out to the XCDs in turn.
    const bool deal = GROUPED && R.ids;
    if (GROUPED && !deal) mtiles = R.tiles[-1];
    const int total = mtiles * ntiles * split.parts, run = (total + 7) / 8, id = deal ? (int)blockIdx.x : (blockIdx.x & 7) * run + (blockIdx.x >> 3);
    if ((!deal && (int)(blockIdx.x >> 3) >= run) || id >= total) return;
    const int part = id % split.parts, tile = id / split.parts;
    const int mt0 = GROUPED ? tile / ntiles : tile % mtiles, nt0 = GROUPED ? tile % ntiles : tile / mtiles;
    __shared__ int slots[GROUPED ? MT * 16 : 1];
    int first, count, e = 0;
    if (GROUPED) {
        const TileRows o = tile_rows<MT * 16>(R, mt0, experts, slots);
        e = o.e, first = o.first, count = o.count;
        if (count == 0) return;
    } else
        first = mt0 * MT * 16, count = min(MT * 16, R.M - first);
    const int col0 = (nt0 * NV + wv) * NT;   // first row tile of W
    f32x4 acc[NW][NT][MT];
#pragma unroll
    for (int q = 0; q < NW; q++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int m = 0; m < MT; m++) acc[q][n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    int top[NW][NT];
#pragma unroll
    for (int q = 0; q < NW; q++)
#pragma unroll
        for (int n = 0; n < NT; n++) top[q][n] = 0;
    if (!GROUPED || e < experts) {
        const int at_k = (int)threadIdx.x % PR * U;
        const T *row[NL];   // rows past the last repeat it and are not stored
#pragma unroll
        for (int u = 0; u < NL; u++) {
            const int i = min(u * (NTH / PR) + (int)threadIdx.x / PR, count - 1);
            long long at;
            if (GROUPED) {
                const int slot = slots[i];
                at = slot / R.S * R.ldt + slot % R.S * R.lds;
            } else
                at = (long long)(first + i) * R.ldt;
            row[u] = (const T *)R.A + at + at_k;
        }
        const u32x4 *wc[NW][NT];   // uniform: the lane is added to each load's offset
        const uint8_t *ws[NW][NT], *tops[NW * NT];
#pragma unroll
        for (int q = 0; q < NW; q++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const Mx4View &V = q ? G : W;
                const long long t = (long long)e * W.rt + min(col0 + n, W.rt - 1);
                wc[q][n] = reinterpret_cast<const u32x4 *>(V.codes) + t * W.kc * 64;
                ws[q][n] = V.scales + t * W.kg * 256;
                tops[q * NT + n] = V.top + (t * 16 + r) * W.kt;
            }
        if (P == 1) row_tops<NW * NT>(tops, W.kt, &top[0][0]);
        const int whole = W.K / 128;
        const int c1 = (int)((long long)whole * part / split.parts), end = (int)((long long)whole * (part + 1) / split.parts);
        u32x4 w[D][NW][NT];
        unsigned s[D][NW][NT];
        TU raw[D][NL];
        auto fetch_weights = [&](int c, int d) {
#pragma unroll
            for (int q = 0; q < NW; q++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    w[d][q][n] = __builtin_nontemporal_load(wc[q][n] + (long long)c * 64 + (unsigned)lane);
                    s[d][q][n] = (ws[q][n] + (c / 4 * 256 + c % 4))[(unsigned)lane * 4];
                }
        };
        auto fetch = [&](int c, int d) {   // chunk c to the registers of place d
            fetch_weights(c, d);
#pragma unroll
            for (int u = 0; u < NL; u++) raw[d][u] = *reinterpret_cast<const TU *>(row[u] + c * 128);
        };
        auto stage = [&](int d, int buf) {   // the rows in place d to LDS
#pragma unroll
            for (int u = 0; u < NL; u++) {
                const int m = u * (NTH / PR) + threadIdx.x / PR;
                G9_LDS unsigned char *at = (G9_LDS unsigned char *)smem + buf * P * PLANE + m * 256 + (((at_k >> 3) ^ swizzle(m)) << 4) + (at_k & 7) * 2;
                typename X::template Piece<U> h[P];
                X::template split_unit<U>(raw[d][u], h);
#pragma unroll
                for (int p = 0; p < P; p++) *reinterpret_cast<G9_LDS typename X::template Piece<U> *>(at + p * PLANE) = h[p];
            }
        };
        const int sw_r = swizzle(r);
        // Steps of eight k and one piece: a step's fragments are read (and its weights converted) while the step before it is
        // multiplied. `half` is called half way.
        auto multiply = [&](int d, int buf, auto half) {
            const G9_LDS unsigned char *base = (const G9_LDS unsigned char *)smem + buf * P * PLANE + r * 256;
            float sc[NW][NT];
#pragma unroll
            for (int q = 0; q < NW; q++)
#pragma unroll
                for (int n = 0; n < NT; n++) sc[q][n] = X::scale(s[d][q][n], top[q][n]);
            Frag a[2][MT], b[2][NW][NT];
            auto prepare = [&](int t) {
#pragma unroll
                for (int m = 0; m < MT; m++) a[t & 1][m] = *reinterpret_cast<const G9_LDS Frag *>(base + t % P * PLANE + m * 4096 + (((4 * g + t / P) ^ sw_r) << 4));
                if (t % P == 0)
#pragma unroll
                    for (int q = 0; q < NW; q++)
#pragma unroll
                        for (int n = 0; n < NT; n++) b[t / P & 1][q][n] = X::weights(w[d][q][n][t / P], sc[q][n]);
            };
            prepare(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < 4 * P; t++) {
                if (t + 1 < 4 * P) prepare(t + 1);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int q = 0; q < NW; q++)
#pragma unroll
                        for (int n = 0; n < NT; n++) acc[q][n][m] = X::mfma(b[t / P & 1][q][n], a[t & 1][m], acc[q][n][m]);
                // the next reads first, then a conversion after each matrix instruction
                __builtin_amdgcn_sched_group_barrier(0x100, MT, 0);
#pragma unroll
                for (int j = 0; j < MT * NW * NT; j++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (t == 2 * P - 1) half();
            }
        };
        if (c1 < end) {
            // No load is conditional (past the end the last chunk is loaded again): a wait then leaves all younger loads on their way.
            // A chunk is staged while the one before it is multiplied; the barrier between them is the one that ends that.
#pragma unroll
            for (int d = 0; d < D; d++) fetch(min(c1 + d, end - 1), d);
            int buf = 0;
            stage(0, 0);
            lds_barrier();
            int c = c1;
            for (; c + D < end; c += D) {
#pragma unroll
                for (int d = 0; d < D; d++) {
                    multiply(d, buf, [&] { stage((d + 1) % D, buf ^ 1); });
                    fetch(min(c + d + D, end - 1), d);
                    buf ^= 1;
                    lds_barrier();
                }
            }
#pragma unroll
            for (int d = 0; d < D; d++) {
                if (c + d >= end) break;
                multiply(d, buf, [&] {
                    if (d + 1 < D && c + d + 1 < end) stage((d + 1) % D, buf ^ 1);
                });
                buf ^= 1;
                lds_barrier();
            }
        }
        if (W.K % 128 && part == split.parts - 1) {   // the chunk in which the rows end
            fetch_weights(whole, 0);
            const int k = whole * 128;
#pragma unroll
            for (int u = 0; u < NL; u++)
#pragma unroll
                for (int j = 0; j < U; j++) raw[0][u][j] = k + at_k + j < W.K ? row[u][k + j] : T(0);
            stage(0, 0);
            __syncthreads();
            multiply(0, 0, [] {});
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        int tn[NW][4];
#pragma unroll
        for (int q = 0; q < NW; q++)
#pragma unroll
            for (int j = 0; j < 4; j++) tn[q][j] = __shfl(top[q][n], 4 * g + j);
        const int col = (col0 + n) * 16 + 4 * g;
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int i = m * 16 + r;
            if (i < count) finish4<T, O, GROUPED, GATED>(R, W, split, part, first, slots, i, col, acc[0][n][m], acc[NW - 1][n][m], tn[0], tn[NW - 1]);
        }
    }
}

}  // namespace g9llm
