// Host side of the FP16 GEMM on direct global→LDS loads (hgemm_kernel.h): which products it takes; their tiles and their
// split of K are hgemm_tiles.h's. Part of gemm_kernels.hip: one code object for the GEMM kernels, loaded as a whole with the first of them.
#pragma once
#include "internal.h"
#include "hgemm_kernel.h"
#include "hgemm_tiles.h"
#include <stdlib.h>
#include <string.h>
#include <algorithm>

namespace g9 {
namespace hgl {

template <int I, bool AK, bool BKC, bool EDGE>
static int launch_cfg(hg::Params p, int count, int slices) {
    constexpr HgCfg G = CFG[I];
    p.tiles_m = (p.M + G.BM - 1) / G.BM;
    p.tiles_n = (p.N + G.BN - 1) / G.BN;
    const dim3 block(G.WM * G.WN * 64);
    const unsigned tiles = (unsigned)(p.tiles_m * p.tiles_n);
    if constexpr (EDGE) {
        if (slices > 1 && p.P) {
            p.kper = std::max(((p.K + slices - 1) / slices + KB - 1) / KB * KB, 2 * KB);
            const int ns = (p.K + p.kper - 1) / p.kper;
            hipLaunchKernelGGL((hg::hgemm_kernel<G.BM, G.BN, G.WM, G.WN, KB, G.NS, AK, BKC, G.RA, true, true>),
                               dim3(tiles, (unsigned)ns), block, 0, stream, p);
            G9_HIP(hipGetLastError());
            constexpr int PER = G.BM * G.BN / 512;   // 512 elements of C per wave
            hipLaunchKernelGGL((hg::split_sum<G.BM, G.BN, G.WM, G.WN>), dim3((unsigned)(((long long)tiles * PER + 3) / 4)),
                               dim3(256), 0, stream, p, ns);
            G9_HIP(hipGetLastError());
            return 0;
        }
    }
    hipLaunchKernelGGL((hg::hgemm_kernel<G.BM, G.BN, G.WM, G.WN, KB, G.NS, AK, BKC, G.RA, EDGE>),
                       dim3(tiles, (unsigned)count), block, 0, stream, p);
    G9_HIP(hipGetLastError());
    return 0;
}
template <bool AK, bool BKC>
static int launch_layout(const hg::Params &p, int count, Choice ch, bool whole) {
    if (whole && ch.slices == 1) {
        switch (ch.cfg) {
        case 0: return launch_cfg<0, AK, BKC, false>(p, count, 1);
        case 1: return launch_cfg<1, AK, BKC, false>(p, count, 1);
        case 2: return launch_cfg<2, AK, BKC, false>(p, count, 1);
        }
    }
    switch (ch.cfg) {
    case 0: return launch_cfg<0, AK, BKC, true>(p, count, ch.slices);
    case 1: return launch_cfg<1, AK, BKC, true>(p, count, ch.slices);
    case 2: return launch_cfg<2, AK, BKC, true>(p, count, ch.slices);
    case 5: return launch_cfg<5, AK, BKC, true>(p, count, ch.slices);
    case 6: return launch_cfg<6, AK, BKC, true>(p, count, ch.slices);
    }
    if constexpr (BKC) {
        if (ch.cfg == 3) return launch_cfg<3, AK, BKC, true>(p, count, ch.slices);
    }
    if constexpr (AK) {
        if (ch.cfg == 4) return launch_cfg<4, AK, BKC, true>(p, count, ch.slices);
    }
    G9_FAIL(GEN9BLAS_ERR_UNSUPPORTED, "hgemm: configuration %d for layout A %d B %d", ch.cfg, AK, BKC);
}

}  // namespace hgl

// FP16 products on the direct global→LDS kernel. False, with nothing launched, for those it does not take; otherwise
// *rc is the launch's status.
// The kernel takes operands at 4-byte alignment with even row (and batch) strides, which its direct copies need, and
// more than one k-step of k (exactly one when no operand row ends inside a 16-byte chunk): the k-step it takes through
// registers needs a direct one beside it. Lane offsets inside a tile are 32-bit (lane_span). GEN9BLAS_HGEMM=generic
// forces the general kernel; a forced split-K (GEN9BLAS_SPLITK) leaves it the products that are whole 128×128 tiles.
static bool launch_hgemm_tiles(const GemmCall &c, int *rc) {
    using namespace hgl;
    static const bool generic = [] {
        const char *e = getenv("GEN9BLAS_HGEMM");
        return e && !strcmp(e, "generic");
    }();
    const bool batch = c.count > 1;
    if (generic || c.count > 65535 || c.lda % 2 || c.ldb % 2 || (uintptr_t)c.A % 4 || (uintptr_t)c.B % 4 ||
        (batch && (c.sA % 2 || c.sB % 2)) || std::min(c.lda, c.ldb) < 8)
        return false;
    if (lane_span(!c.tA, c.lda * 2, c.M, KB) >= (1LL << 32) || lane_span(c.tB, c.ldb * 2, c.N, KB) >= (1LL << 32)) return false;
    if (c.K < KB || (c.K == KB && ((c.tA && c.M % 8) || (!c.tB && c.N % 8)))) return false;
    // whole: nothing to check or mask, 16-byte stores
    const auto al16 = [&](const void *x, long long ld, long long s) {
        return (uintptr_t)x % 16 == 0 && ld % 8 == 0 && (!batch || s % 8 == 0);
    };
    const bool aligned = al16(c.A, c.lda, c.sA) && al16(c.B, c.ldb, c.sB) && al16(c.C, c.ldc, c.sC);
    const bool whole128 = aligned && c.M % 128 == 0 && c.N % 128 == 0 && c.K % KB == 0;
    if (splitk_forced() >= 0 && !whole128) return false;
    // the work space of split products is reserved at its bound with the first product here, so that no later call waits
    // for queued work to let it grow
    void *P = nullptr;
    size_t work = 0;
    if (!batch && splitk_forced() < 0) P = splitk_workspace(&work);
    const Choice ch = choose({c.M, c.N, c.K, c.count, c.ldc, c.tA, c.tB}, work, num_cus);
    const HgCfg &g = CFG[ch.cfg];
    if (tiles_of(g, c.M, c.N) > 0x7fffffffLL) return false;
    const bool whole = aligned && c.M % g.BM == 0 && c.N % g.BN == 0 && c.K % KB == 0;

    hg::Params p;
    p.A = reinterpret_cast<const hg::f16 *>(c.A);
    p.B = reinterpret_cast<const hg::f16 *>(c.B);
    p.C = reinterpret_cast<hg::f16 *>(c.C);
    p.lda = c.lda; p.ldb = c.ldb; p.ldc = c.ldc;
    p.sA = batch ? c.sA : 0; p.sB = batch ? c.sB : 0; p.sC = batch ? c.sC : 0;
    p.M = c.M; p.N = c.N; p.K = c.K;
    p.tiles_m = p.tiles_n = 0;
    p.P = reinterpret_cast<float *>(P);
    p.alpha = (float)c.alpha;
    p.beta = (float)c.beta;
    if (c.tA) *rc = c.tB ? launch_layout<false, true>(p, c.count, ch, whole) : launch_layout<false, false>(p, c.count, ch, whole);
    else *rc = c.tB ? launch_layout<true, true>(p, c.count, ch, whole) : launch_layout<true, false>(p, c.count, ch, whole);
    return true;
}

}  // namespace g9
