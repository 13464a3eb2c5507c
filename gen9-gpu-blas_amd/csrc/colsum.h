// Sums over rows for the gradients of a bias or a norm's weights: kernels leave the sums of blocks of rows in a work buffer, and
// this adds the blocks in a fixed order, so results do not vary from call to call.
#pragma once
#include "llm.h"
#include <algorithm>

namespace g9llm {

// out[n] (+)= Σ_b parts[b·ld + n], and, blockIdx.y = 1, out2 of the columns `second` behind: 64 columns a workgroup, 16 threads a column,
// each with every sixteenth block.
static __global__ void __launch_bounds__(1024) column_sums_kernel(const float *__restrict__ parts, long long blocks, int N, int second, long long ld, float *out, float *out2, int accumulate) {
    __shared__ float part[16][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6, n = blockIdx.x * 64 + c;
    if (blockIdx.y) parts += second, out = out2;
    if (!out) return;
    float s[4] = {};
    if (n < N) {
        long long b = r;
        for (; b + 48 < blocks; b += 64)
#pragma unroll
            for (int i = 0; i < 4; i++) s[i] += parts[(b + 16 * i) * ld + n];
        for (; b < blocks; b += 16) s[0] += parts[b * ld + n];
    }
    part[r][c] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (r || n >= N) return;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) sum += part[i][c];
    out[n] = accumulate ? out[n] + sum : sum;
}
static int column_sums(const float *parts, long long blocks, int N, long long ld, float *out, float *out2, int accumulate) {
    constexpr long long MOST = 1 << 27;   // columns of a launch, which indexes 2^32 threads
    for (long long n = 0; n < N; n += MOST) {
        const int count = (int)std::min(N - n, MOST);
        hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)cdiv(count, 64), out2 ? 2 : 1), dim3(1024), 0, stream, parts + n, blocks, count, N, ld,
                           out ? out + n : nullptr, out2 ? out2 + n : nullptr, accumulate);
        G9_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace g9llm
