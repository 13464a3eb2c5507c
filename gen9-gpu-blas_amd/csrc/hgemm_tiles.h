// FP16 products on direct global→LDS loads (hgemm_kernel.h): their tiles and their split of K.
//
// Tile configurations come from sweeps on MI355X with N(0,1) FP16 inputs, timed after 1.5 s of the same load (the clock
// settles under the board's power limit; shorter runs see its ramp), every variant bit-exact on small integers:
// - 256×256 tiles, 8 waves of 128×64 (2×4), two stages of 64 k. n = 4096 NN 1314-1324 TFLOP/s (8 waves of 64×128:
//   1276-1286; 4 waves of 128×128: 1243-1246, at 2.03 GHz against 1.79-1.81; the same 8 waves on 32x32x16 MFMAs:
//   1166-1176); TN 1249, NT 1339, TT 1267 (32x32x16: 1180-1188);
// - 128×128, 8 waves of 64×32 (2×4), three stages. n = 2048 NN 835 (4 waves of 64×64 with 3 or 4 stages: 798-807;
//   32x32x16 tiles: 795), NT 845 (767), TN and TT 800-804 (800-802);
// - 64×64, 4 waves of 32×32, three stages, fragments read one k-step ahead: n = 1024 NT 399.9 (four stages 390.6, two
//   303.6, no read-ahead 378.1), NN 400.7 (its 64-wide mn-contiguous B rows swizzled by mnswz). Before them 32×128
//   tiles, NN 382.8; 128×128 tiles for a transposed A, TN 212.6 → 365.5, TT 215.3 → 393.1. Time per call against K at
//   M = N = 1024 is about 2-3 µs plus 0.26 µs per k-step of 64: the k-step's latency chain sets the rate;
// - 256×192 (192×256), 8 waves of 64×96 (96×64), two stages, and 256×128 (128×256), 8 waves of 64×64, three stages, for
//   tile counts that leave the larger tiles' last round, or the only one, part empty (µs): 1000×11008×4096 NT 94.5 on
//   232 tiles of 256×192 against 100.7 on 172 of 256×256, 114 on 688 of 128×128 and 109 on 344 of 256×128; 2504³ NT 60.4
//   on 200 of 128×256 against 66.2 on 400 of 128×128. A 192-wide operand must be k-contiguous.
#pragma once
#include <stddef.h>
#include <algorithm>
#include <cmath>

namespace g9 {

// Bytes that the direct copies' lane offsets reach over inside a tile of at most 256 rows: the rows of a k-contiguous
// operand of MN rows, the k rows of a k-step otherwise (ldb: row stride in bytes). They are 32-bit.
static long long lane_span(bool kc, long long ldb, int MN, int kb) { return (kc ? std::min(256, MN) : kb) * ldb; }

namespace hgl {

constexpr int KB = 64;   // k per k-step
// For choose(): ns, time per k of a round of one tile per CU on the whole chip; fix, the rest of a round (µs); st, µs per MB
// of C stored
struct HgCfg { int BM, BN, WM, WN, NS; bool RA; double ns, fix, st; };
constexpr HgCfg CFG[] = {{256, 256, 2, 4, 2, false, 25, 3.1, 0.062}, {128, 128, 2, 4, 3, false, 8.1, 1.8, 0.037},
                         {64, 64, 2, 2, 3, true, 3.3, 1.8, 0}, {256, 192, 4, 2, 2, false, 22, 2.1, 0.064},
                         {192, 256, 2, 4, 2, false, 22, 2.1, 0.064}, {256, 128, 4, 2, 3, false, 13.07, 3, 0.044},
                         {128, 256, 2, 4, 3, false, 13, 3, 0.044}};
constexpr int NCFG = sizeof CFG / sizeof CFG[0];

// C (M×N, row stride ldc) = op(A)·op(B), `count` of them
struct Size { int M, N, K, count; long long ldc; int tA, tB; };

static long long tiles_of(const HgCfg &g, int M, int N) { return (long long)((M + g.BM - 1) / g.BM) * ((N + g.BN - 1) / g.BN); }

struct Choice { int cfg, slices; };
// The configuration and number of K slices with the smallest estimated time (µs): a launch; rounds of one tile per CU
// (64×64: two share a CU, one alone takes two thirds of their time), each a fixed part and the tile's time per k, less where
// part of the chip idles (the board's power limit leaves the rest a higher clock); C written by the larger tiles, which
// costs most where its rows are not whole 128-byte lines; for slices, the second kernel, its pass over each slice, and the
// FP32 sums written and read.
// The constants are a fit to the order of 392 products (K 64 to 11008, 17 to 20000 rows, batches, whole and ragged, NN /
// NT / TN), each timed with every configuration and 1-16 slices on operands in the last-level cache and rotated beyond it:
// by the geometric mean of both the choice is 0.6 % from the fastest on average, and within 22 % for all. A few (µs,
// in the cache and beyond it, chosen / others): 48×4096×4096 NT 64×64 in 4 slices 10.7 and 12.7 / unsplit 21 and 23;
// 600×4096×11008 128×256 in 3 slices 74 / 128×128 unsplit 103; 256×1024×1024 64×64 5.4 and 8.2 / in 3 slices 7.5 and 8.5;
// 1280³ 64×64 9.1 and 11.7 / 128×128 11.3 and 14.4; 5000×5000×64 64×64 or 128×128 27 and 31 / 256×256 41 and 48. Slices hold
// at least 256 k and fit the `work` bytes of the split-K work space.
static Choice choose(const Size &c, size_t work, int num_cus) {
    static constexpr int SLICES[] = {1, 2, 3, 4, 6, 8, 12, 16};
    const double mn = (double)c.M * c.N, c_mb = 2e-6 * c.count * mn * (c.ldc % 64 ? 7 : 1);
    Choice best{0, 1};
    double t_best = 1e30;
    for (int i = 0; i < NCFG; i++) {
        const HgCfg &g = CFG[i];
        if ((g.BN == 192 && !c.tB) || (g.BM == 192 && c.tA)) continue;
        const long long tiles = tiles_of(g, c.M, c.N) * c.count;
        for (const int s : SLICES) {
            const int kper = ((c.K + s - 1) / s + KB - 1) / KB * KB, ns = (c.K + kper - 1) / kper;
            if (s > 1 && (kper < 256 || tiles * s > 3LL * num_cus ||
                          (size_t)(ns * tiles) * g.BM * g.BN * sizeof(float) > work)) break;
            const bool shared = g.BM == 64;
            const double per_cu = (double)(tiles * ns) / num_cus, rounds = std::ceil(per_cu);
            const double load = 0.8 * rounds + 0.2 * per_cu;
            const double t = 2.8 + g.ns * 1e-3 * kper * (shared ? std::max(1.3, load) : load) +
                             g.fix * (shared ? std::max(1.0, per_cu / 2) : rounds) +
                             (ns > 1 ? 1.8 + 0.46 * ns + ns * mn * 8 / 9.2e6 : g.st * c_mb);
            if (t < t_best) {
                t_best = t;
                best = Choice{i, ns};
            }
        }
    }
    return best;
}

}  // namespace hgl
}  // namespace g9
