// FP32 products on direct global→LDS loads (sgemm_kernel.h): their tiles and their split of K.
//
// Tile configurations, with rates on MI355X (TFLOP/s, sustained): 128×256, 8 waves of 64×64, two stages, sums blocked per
// 128 k: n = 4096 NN 144.9, NT 144.3, 8192×8192×2048 144.1 (three stages 142.6; blocks of 32 k 134.3, 64 k 140.3, 256 k
// 142.6; 256×128 tiles 142.7). 128×128, 8 waves of 64×32, three stages: n = 2048 133-134 (4 waves of 64×64 129.7).
// 64×64, 4 waves of 32×32, four stages, sums blocked per 256 k: n = 2048 137, n = 1024 102.6 (three stages 94.0, six 93.0,
// eight 92.2; 128-k blocks 101.9, 32-k 90.9). 64×128 and 128×64, 4 waves of 32×64 (64×32), three stages:
// 2386×1512×1920 120.5 µs against 121.1 on 64×64 and 122.1 on 128×128 tiles, 3000×3000×150 42.6 against 43.1 and 46.5.
#pragma once
#include <stddef.h>
#include <algorithm>
#include <cmath>

namespace g9 {
namespace sgl {

constexpr int KB = 32;   // k per k-step
// ns: time per k of a 64×64 share of the tile, for cost(); per_cu: workgroups that share a CU
struct SgCfg { int BM, BN, WM, WN, NS, BLK; double ns; int per_cu; };
constexpr SgCfg CFG[] = {{128, 256, 2, 4, 2, 4, 14.4, 1}, {128, 128, 2, 4, 3, 4, 14.8, 1}, {64, 64, 2, 2, 4, 8, 14.8, 2},
                         {64, 128, 2, 2, 3, 4, 14.8, 2}, {128, 64, 2, 2, 3, 4, 14.8, 2}};
constexpr int NCFG = sizeof CFG / sizeof CFG[0];
struct Choice { int cfg, slices; double us; };
struct Size { int M, N, K, count; };   // C (M×N) = op(A)·op(B), `count` of them

static int slices_of(int K, int s, int &kper) {
    kper = std::max(((K + s - 1) / s + KB - 1) / KB * KB, 2 * KB);
    return (K + kper - 1) / kper;
}
// Estimated time (µs) of `tiles` tiles of a configuration in ns slices of kper k: the launch, the most loaded CU's tiles at
// the matrix cores' rate, a fixed part for each round of tiles that share a CU, and for slices the second kernel and
// their sums written and read. Constants fitted to 29 products (K 100 to 20000, 100 to 8000 rows, batches, whole and
// ragged, every layout), timed with every configuration and 1-24 slices: the choice is the fastest or within 2 % of it for
// 27 of them, within 7 % for all. A few (µs, chosen / others): 500³ 64×64 in 3 slices 10.2 / unsplit 12.1; 130×130×5000
// 64×64 in 16-24 slices 16.9 / in 4 24; 64 × 256³ 128×128 24.8 / 64×64 27.4; 245 × 144×64×264 64×64 25.5 / 128×128 48.5.
static double cost(const SgCfg &g, long long tiles, int kper, int ns, int num_cus) {
    const double per_cu = (double)(tiles * ns) / num_cus, area = (double)g.BM * g.BN / 4096;
    double t = 5.4 + std::max(1.0, std::ceil(per_cu)) * area * g.ns * 1e-3 * kper + 3.4 * std::ceil(per_cu / g.per_cu);
    if (ns > 1) t += 0.8 + (double)(ns * tiles) * g.BM * g.BN * 8 / 1e7;
    return t;
}
// The cheapest configuration and split of K into slices that fit `work` bytes; tri: the tiles of a triangle of side M
// (square tiles only); big: 128×256 tiles may be taken (their edge-capable variant would need more registers than a wave
// has).
static Choice choose(const Size &c, size_t work, bool tri, bool big, int num_cus) {
    static constexpr int SLICES[] = {1, 2, 3, 4, 6, 8, 12, 16, 24};
    Choice best{2, 1, 1e30};
    for (int i = 0; i < NCFG; i++) {
        const SgCfg &g = CFG[i];
        // a triangle that no whole tiles fill: 128×128 tiles lose half of each on the diagonal, and on this kernel they
        // were slower throughout (2000×200 22.1 µs against 20.0, 5000×160 50.8 against 40.3)
        if ((tri && (g.BM != g.BN || (g.BM == 128 && c.M % 64))) || (i == 0 && !big)) continue;
        const long long tm = (c.M + g.BM - 1) / g.BM, tn = (c.N + g.BN - 1) / g.BN;
        const long long tiles = (tri ? tm * (tm + 1) / 2 : tm * tn) * c.count;
        for (const int s : SLICES) {
            int kper;
            const int ns = s == 1 ? 1 : slices_of(c.K, s, kper);
            if (s == 1) kper = (c.K + KB - 1) / KB * KB;
            if (s > 1 && (i == 0 || kper < 4 * KB || tiles * s > 5LL * num_cus ||
                          (size_t)(ns * tiles) * g.BM * g.BN * sizeof(float) > work)) break;
            const double t = cost(g, tiles, kper, ns, num_cus);
            if (t < best.us) best = Choice{i, ns, t};
        }
    }
    return best;
}

}  // namespace sgl
}  // namespace g9
