// 16-bit activations times packed int4 weights with a scale per group of K: D[m][n] = round16(sum_g scale[n][g] *
// sum_{k in g} x[m][k] * B[n][k] + bias[n]).
#pragma once
#include "qm_float16.hpp"

namespace qm {

struct GroupedArgs {
    const uint16_t *x;  // [M, K], rows `x_stride` elements apart
    const uint8_t *B;   // [N, K/2]
    const void *scale;  // [N, groups]
    const uint16_t *bias;
    uint16_t *D;
    long long x_stride;
    int M, N, K, group, groups;
};

// Any even K at any address: a wave to a column and four rows, a lane to a byte of B at a time, two elements of each
// row with it. Every scaled element goes into the sum by itself.
constexpr int GROUPED_ROWS = 4;
template <int T, int S>
__global__ __launch_bounds__(256) void gemm_grouped_any_kernel(const GroupedArgs p)
{
    const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= p.N) return;
    const uint8_t *const b = p.B + (size_t)n * (p.K / 2);
    for (long long m0 = (long long)blockIdx.y * GROUPED_ROWS; m0 < p.M; m0 += (long long)gridDim.y * GROUPED_ROWS) {
        float sum[GROUPED_ROWS] = {};
        for (int j = lane; j < p.K / 2; j += 64) {
            const float s = element<S>(p.scale, (size_t)n * p.groups + 2 * j / p.group);
            const int byte = (int8_t)b[j];
            const float lo = (float)((int)((uint32_t)byte << 28) >> 28) * s, hi = (float)(byte >> 4) * s;
#pragma unroll
            for (int r = 0; r < GROUPED_ROWS; ++r) {
                const uint16_t *const x = p.x + (m0 + r < p.M ? m0 + r : m0) * p.x_stride + 2 * j;
                sum[r] = __builtin_fmaf(float_of<T>(x[1]), hi, __builtin_fmaf(float_of<T>(x[0]), lo, sum[r]));
            }
        }
#pragma unroll
        for (int r = 0; r < GROUPED_ROWS; ++r) {
            float v = sum[r];
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
            if (lane == 0 && m0 + r < p.M) p.D[(m0 + r) * p.N + n] = round16<T>(p.bias != nullptr ? v + float_of<T>(p.bias[n]) : v);
        }
    }
}

}  // namespace qm
