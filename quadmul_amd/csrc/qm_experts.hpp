// 16-bit activations times the packed int4 weights of each token's experts. Choice j of token t is slot t * top_k + j: its row of x times
// the matrix of its expert. The definitions are those of include/qm_abi.h.
#pragma once
#include "qm_grouped.hpp"

namespace qm {

// What becomes of a slot's products: rounded, with the bias (and zeros where the expert is none of these); the first half of the columns as gates of
// the second, rounded; as they are, to be added up by weight.
enum ExpertsOut { EXPERTS_PLAIN, EXPERTS_GATED, EXPERTS_PART };

struct ExpertsArgs {
    const uint16_t *x;
    long long x_token, x_choice;  // in elements, between tokens and between choices
    const int *chosen;            // [slots]
    const uint8_t *B;             // [experts, N, K/2]
    const void *scale;            // [experts, N, groups]
    const uint16_t *bias;         // [experts, N] or null
    void *out;                    // [slots, N], [slots, N/2] 16-bit, or [slots, N] float
    int slots, top_k, experts, N, K, group, groups;
};
__device__ __forceinline__ const uint16_t *row_of(const ExpertsArgs &p, const int slot)
{
    const int t = slot / p.top_k;
    return p.x + t * p.x_token + (slot - t * p.top_k) * p.x_choice;
}
// silu(gate) * value
__device__ __forceinline__ float gated(const float gate, const float value) { return gate / (1.0f + __expf(-gate)) * value; }

// Any even K at any address: a wave to a slot and a column (two columns where one gates the other), a lane to a byte of B at a time.
template <int T, int S, int OUT>
__global__ __launch_bounds__(256) void experts_any_kernel(const ExpertsArgs p)
{
    const int lane = threadIdx.x & 63, columns = OUT == EXPERTS_GATED ? p.N / 2 : p.N;
    for (long long slot = blockIdx.y; slot < p.slots; slot += gridDim.y) {
        const int expert = p.chosen[slot];
        const bool none = (unsigned)expert >= (unsigned)p.experts;
        if (none && OUT != EXPERTS_PLAIN) continue;
        const uint16_t *const x = row_of(p, (int)slot);
        for (long long n = blockIdx.x * 4 + (threadIdx.x >> 6); n < columns; n += (long long)gridDim.x * 4) {
            float sum[2] = {};
            if (!none) {
#pragma unroll
                for (int half = 0; half < (OUT == EXPERTS_GATED ? 2 : 1); ++half) {
                    const size_t row = (size_t)expert * p.N + n + half * columns;
                    const uint8_t *const b = p.B + row * (p.K / 2);
                    float v = 0.0f;
                    for (int j = lane; j < p.K / 2; j += 64) {
                        const float s = element<S>(p.scale, row * p.groups + 2 * j / p.group);
                        const int byte = (int8_t)b[j];
                        const float lo = (float)((int)((uint32_t)byte << 28) >> 28) * s, hi = (float)(byte >> 4) * s;
                        v = __builtin_fmaf(float_of<T>(x[2 * j + 1]), hi, __builtin_fmaf(float_of<T>(x[2 * j]), lo, v));
                    }
#pragma unroll
                    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
                    sum[half] = v;
                }
            }
            if (lane != 0) continue;
            if (OUT == EXPERTS_PART) static_cast<float *>(p.out)[slot * p.N + n] = sum[0];
            else if (OUT == EXPERTS_GATED) static_cast<uint16_t *>(p.out)[slot * columns + n] = round16<T>(gated(sum[0], sum[1]));
            else static_cast<uint16_t *>(p.out)[slot * p.N + n] = none ? 0 : round16<T>(p.bias != nullptr ? sum[0] + float_of<T>(p.bias[(size_t)expert * p.N + n]) : sum[0]);
        }
    }
}

// y[t] = sum over a token's choices, in their order, of weight times product.
template <int T>
__global__ __launch_bounds__(256) void experts_sum_kernel(const float *part, const int *chosen, const float *weights, uint16_t *y, const int tokens, const int top_k, const int experts, const int N)
{
    const size_t all = (size_t)tokens * N;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        const size_t t = i / N, n = i - t * N;
        float v = 0.0f;
        for (int j = 0; j < top_k; ++j) {
            const size_t slot = t * top_k + j;
            if ((unsigned)chosen[slot] < (unsigned)experts) v = __builtin_fmaf(weights[slot], part[slot * N + n], v);
        }
        y[i] = round16<T>(v);
    }
}

}  // namespace qm
