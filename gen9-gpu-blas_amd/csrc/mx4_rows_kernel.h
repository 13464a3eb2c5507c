// Products of few rows with MX4 weights (decode): the weights are read once, straight into the registers that multiply them.
#pragma once
#include "mx4_gemm_kernel.h"

namespace g9llm {

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

// The end of a row's four columns col .. col + 3 (y: the sum with W, z: with the gate): to C, or as a part's sums.
template <class T, class O, bool GROUPED, bool GATED>
__device__ __forceinline__ void finish4(const Rows &R, const Mx4View &W, const Split &split, int part, int first, int i, int col, f32x4 y, f32x4 z, const int *ty,
                                        const int *tz) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        y[j] = Act<T>::finish(y[j], ty[j]);
        if (GATED) z[j] = Act<T>::finish(z[j], tz[j]);
    }
    if (split.parts > 1) {
        if (col >= W.rows) return;   // ld is whole column tiles
        float *p = split.sums + ((long long)part * (GATED ? 2 : 1) * split.rows + first + i) * split.ld + col;
        *reinterpret_cast<f32x4 *>(p) = y;
        if (GATED) *reinterpret_cast<f32x4 *>(p + split.rows * split.ld) = z;
        return;
    }
    O *c;
    if (GROUPED) {
        const int slot = R.order[first + i];
        c = (O *)R.C + slot / R.S * R.ldct + slot % R.S * R.ldcs;
    } else
        c = (O *)R.C + (long long)(first + i) * R.ldct;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (col + j < W.rows) c[col + j] = (O)(GATED ? y[j] * silu(z[j]) : y[j]);
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

// A workgroup has WN × WK waves (WN · WK = 4): WN side by side in n, each 16·NT columns (gated: of W and of the gate) of MT·16
// rows, and WK along k; `split` workgroups share the k of a tile. Weights and rows of the next D chunks of 128 k are
// on their way in registers. Lane 16g + r multiplies columns' row r of each weight tile, activations' row r.
template <class T, class O, int MT, int NT, int WN, int D, bool GROUPED, bool GATED>
__global__ void __launch_bounds__(256) mx4_gemm_rows_kernel(Rows R, Mx4View W, Mx4View G, int experts, int ntiles, Split split) {
    typedef Act<T> X;
    typedef typename X::Frag Frag;
    constexpr int NW = GATED ? 2 : 1, WK = 4 / WN, NA = NW * NT * MT;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int part = blockIdx.x % split.parts, tile = blockIdx.x / split.parts;
    const int mt0 = tile / ntiles, nt0 = tile % ntiles;
    int first, count, e = 0;
    if (GROUPED) {
        if (mt0 >= R.tiles[-1]) return;
        e = R.tiles[2 * mt0], first = R.tiles[2 * mt0 + 1];
        count = min(MT * 16, R.off[e + 1] - first);
    } else
        first = mt0 * MT * 16, count = min(MT * 16, R.M - first);
    const int col0 = (nt0 * WN + wv % WN) * NT;   // first row tile of W
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
        const T *row[MT];   // rows past the last repeat it and are not stored
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int i = first + min(m * 16 + r, count - 1);
            long long at;
            if (GROUPED) {
                const int slot = R.order[i];
                at = slot / R.S * R.ldt + slot % R.S * R.lds;
            } else
                at = (long long)i * R.ldt;
            row[m] = (const T *)R.A + at + g * 32;
        }
        const u32x4 *wc[NW][NT];
        const uint8_t *ws[NW][NT];
#pragma unroll
        for (int q = 0; q < NW; q++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const Mx4View &V = q ? G : W;
                const long long t = (long long)e * W.rt + min(col0 + n, W.rt - 1);
                wc[q][n] = reinterpret_cast<const u32x4 *>(V.codes) + t * W.kc * 64 + lane;
                ws[q][n] = V.scales + t * W.kg * 256 + lane * 4;
                if (X::P == 1) top[q][n] = row_top(V.top + (t * 16 + r) * W.kt, W.kt);
            }
        const int ways = split.parts * WK, way = part * WK + wv / WN, whole = W.K / 128;
        const int c1 = (int)((long long)whole * way / ways), end = (int)((long long)whole * (way + 1) / ways);
        u32x4 w[D][NW][NT];
        unsigned s[D][NW][NT];
        Row32<T> a[D][MT];
        auto fetch_weights = [&](int c, int d) {
#pragma unroll
            for (int q = 0; q < NW; q++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    w[d][q][n] = __builtin_nontemporal_load(wc[q][n] + (long long)c * 64);
                    s[d][q][n] = ws[q][n][c / 4 * 256 + c % 4];
                }
        };
        auto fetch = [&](int c, int d) {   // chunk c to the registers of place d
            fetch_weights(c, d);
#pragma unroll
            for (int m = 0; m < MT; m++) a[d][m].load(row[m] + c * 128);
        };
        auto multiply = [&](int d) {
            Frag f[MT][4][X::P];
#pragma unroll
            for (int m = 0; m < MT; m++) a[d][m].fragments(f[m]);
#pragma unroll
            for (int q = 0; q < NW; q++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const float sc = X::scale(s[d][q][n], top[q][n]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const Frag b = X::weights(w[d][q][n][i], sc);
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int p = 0; p < X::P; p++) acc[q][n][m] = X::mfma(b, f[m][i][p], acc[q][n][m]);
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
#pragma unroll
            for (int m = 0; m < MT; m++) a[0][m].load_tail(row[m] - g * 32, whole * 128 + g * 32, W.K);
            multiply(0);
        }
    }
    // the sums of the waves along k, in their order
    if (WK > 1) {
        __shared__ f32x4 sums[(WK - 1) * WN * NA * 64];
        if (wv >= WN) {
#pragma unroll
            for (int i = 0; i < NA; i++) sums[((wv - WN) * NA + i) * 64 + lane] = acc[i / (NT * MT)][i / MT % NT][i % MT];
        }
        __syncthreads();
        if (wv < WN) {
#pragma unroll
            for (int k = 1; k < WK; k++)
#pragma unroll
                for (int i = 0; i < NA; i++) acc[i / (NT * MT)][i / MT % NT][i % MT] += sums[(((k - 1) * WN + wv) * NA + i) * 64 + lane];
        }
    }
    if (wv >= WN) return;
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
            if (i < count) finish4<T, O, GROUPED, GATED>(R, W, split, part, first, i, col, acc[0][n][m], acc[NW - 1][n][m], tn[0], tn[NW - 1]);
        }
    }
}

// A barrier for what waves pass each other in LDS: their loads from memory stay on their way (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    g9::wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// 8 waves side by side in n, each 16·NT columns (gated: of W and of the gate) of MT·16 rows. The rows of each 128 k are taken
// apart once for the whole workgroup, into FP16 or BF16 planes in LDS (two buffers; 16-byte piece q of row m at q ^ (m & 15)):
// thread t loads four k at a time, 32 threads to a row. Weights and rows of the next D chunks are on their way in registers;
// both, as loads return in order and the wait for the nearest rows would be a wait for all older weights too.
template <class T, class O, int MT, int NT, int D, bool GROUPED, bool GATED>
__global__ void __launch_bounds__(512) mx4_gemm_few_kernel(Rows R, Mx4View W, Mx4View G, int experts, int ntiles, Split split) {
    typedef Act<T> X;
    typedef typename X::Frag Frag;
    typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    constexpr int NW = GATED ? 2 : 1, P = X::P, PLANE = MT * 4096;
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * P * PLANE];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int part = blockIdx.x % split.parts, tile = blockIdx.x / split.parts;
    const int mt0 = tile / ntiles, nt0 = tile % ntiles;
    int first, count, e = 0;
    if (GROUPED) {
        if (mt0 >= R.tiles[-1]) return;
        e = R.tiles[2 * mt0], first = R.tiles[2 * mt0 + 1];
        count = min(MT * 16, R.off[e + 1] - first);
    } else
        first = mt0 * MT * 16, count = min(MT * 16, R.M - first);
    const int col0 = (nt0 * 8 + wv) * NT;   // first row tile of W
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
        const int quad = threadIdx.x & 31;
        const T *row[MT];   // rows past the last repeat it and are not stored
#pragma unroll
        for (int u = 0; u < MT; u++) {
            const int i = first + min(u * 16 + (int)(threadIdx.x >> 5), count - 1);
            long long at;
            if (GROUPED) {
                const int slot = R.order[i];
                at = slot / R.S * R.ldt + slot % R.S * R.lds;
            } else
                at = (long long)i * R.ldt;
            row[u] = (const T *)R.A + at;
        }
        const u32x4 *wc[NW][NT];
        const uint8_t *ws[NW][NT];
#pragma unroll
        for (int q = 0; q < NW; q++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const Mx4View &V = q ? G : W;
                const long long t = (long long)e * W.rt + min(col0 + n, W.rt - 1);
                wc[q][n] = reinterpret_cast<const u32x4 *>(V.codes) + t * W.kc * 64 + lane;
                ws[q][n] = V.scales + t * W.kg * 256 + lane * 4;
                if (P == 1) top[q][n] = row_top(V.top + (t * 16 + r) * W.kt, W.kt);
            }
        const int whole = W.K / 128;
        const int c1 = (int)((long long)whole * part / split.parts), end = (int)((long long)whole * (part + 1) / split.parts);
        u32x4 w[D][NW][NT];
        unsigned s[D][NW][NT];
        T4 raw[D][MT];
        auto fetch_weights = [&](int c, int d) {
#pragma unroll
            for (int q = 0; q < NW; q++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    w[d][q][n] = __builtin_nontemporal_load(wc[q][n] + (long long)c * 64);
                    s[d][q][n] = ws[q][n][c / 4 * 256 + c % 4];
                }
        };
        auto fetch = [&](int c, int d) {   // chunk c to the registers of place d
            fetch_weights(c, d);
#pragma unroll
            for (int u = 0; u < MT; u++) raw[d][u] = *reinterpret_cast<const T4 *>(row[u] + c * 128 + quad * 4);
        };
        auto stage = [&](int d, int buf) {   // the rows in place d to LDS
#pragma unroll
            for (int u = 0; u < MT; u++) {
                const int m = u * 16 + (threadIdx.x >> 5);
                G9_LDS unsigned char *at = (G9_LDS unsigned char *)smem + buf * P * PLANE + m * 256 + (((quad >> 1) ^ (m & 15)) << 4) + (quad & 1) * 8;
                unsigned long long h[P];
                X::split4(raw[d][u], h);
#pragma unroll
                for (int p = 0; p < P; p++) *reinterpret_cast<G9_LDS unsigned long long *>(at + p * PLANE) = h[p];
            }
        };
        auto multiply = [&](int d, int buf) {
            const G9_LDS unsigned char *base = (const G9_LDS unsigned char *)smem + buf * P * PLANE + r * 256;
            float sc[NW][NT];
#pragma unroll
            for (int q = 0; q < NW; q++)
#pragma unroll
                for (int n = 0; n < NT; n++) sc[q][n] = X::scale(s[d][q][n], top[q][n]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                Frag b[NW][NT];
#pragma unroll
                for (int q = 0; q < NW; q++)
#pragma unroll
                    for (int n = 0; n < NT; n++) b[q][n] = X::weights(w[d][q][n][i], sc[q][n]);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int p = 0; p < P; p++) {
                        const Frag a = *reinterpret_cast<const G9_LDS Frag *>(base + p * PLANE + m * 4096 + (((4 * g + i) ^ r) << 4));
#pragma unroll
                        for (int q = 0; q < NW; q++)
#pragma unroll
                            for (int n = 0; n < NT; n++) acc[q][n][m] = X::mfma(b[q][n], a, acc[q][n][m]);
                    }
            }
        };
        if (c1 < end) {
            // No load is conditional (past the end the last chunk is loaded again): a wait then leaves all younger loads on their way.
            // Buffer d & 1 (D is even) holds chunk c + d; the barrier before a chunk is multiplied is the one after it was staged.
            static_assert(D % 2 == 0, "two LDS buffers");
#pragma unroll
            for (int d = 0; d < D; d++) fetch(min(c1 + d, end - 1), d);
            stage(0, 0);
            lds_barrier();
            int c = c1;
            for (; c + D < end; c += D) {
#pragma unroll
                for (int d = 0; d < D; d++) {
                    stage((d + 1) % D, (d + 1) & 1);
                    multiply(d, d & 1);
                    fetch(min(c + d + D, end - 1), d);
                    lds_barrier();
                }
            }
#pragma unroll
            for (int d = 0; d < D; d++) {
                if (c + d >= end) break;
                if (d + 1 < D && c + d + 1 < end) stage(d + 1, (d + 1) & 1);
                multiply(d, d & 1);
                lds_barrier();
            }
        }
        if (W.K % 128 && part == split.parts - 1) {   // the chunk in which the rows end
            fetch_weights(whole, 0);
            const int k = whole * 128 + quad * 4;
#pragma unroll
            for (int u = 0; u < MT; u++)
#pragma unroll
                for (int j = 0; j < 4; j++) raw[0][u][j] = k + j < W.K ? row[u][k + j] : T(0);
            stage(0, 0);
            __syncthreads();
            multiply(0, 0);
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
            if (i < count) finish4<T, O, GROUPED, GATED>(R, W, split, part, first, i, col, acc[0][n][m], acc[NW - 1][n][m], tn[0], tn[NW - 1]);
        }
    }
}

}  // namespace g9llm
