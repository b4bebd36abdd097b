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
    int chunk;                // blocks of 32 of K
    // The slots sorted by expert, cut into tiles of rows: their expert, where they begin in `order` and how many they are. After
    // those of the last expert, as number `experts`, slots that have none.
    const int *order, *tiles, *count;  // [slots], [tiles][4], [1]
};
__device__ __forceinline__ const uint16_t *row_of(const ExpertsArgs &p, const int slot)
{
    const int t = slot / p.top_k;
    return p.x + t * p.x_token + (slot - t * p.top_k) * p.x_choice;
}
// silu(gate) * value
__device__ __forceinline__ float gated(const float gate, const float value) { return gate / (1.0f + __expf(-gate)) * value; }

// The slots by expert, and tiles of up to `rows` of each expert's. One workgroup: counts, their sums, places, all in the LDS. Which place of its expert's a slot gets is
// chance, and no result depends on it: every row of a tile is summed by itself.
constexpr int EXPERTS_SORTED = 4096;  // experts at most
__global__ __launch_bounds__(1024) void experts_sort_kernel(const int *chosen, const int slots, const int experts, const int rows, int *order, int *tiles, int *count)
{
    extern __shared__ int bins[];  // [experts + 1]
    __shared__ int sums[2][16];
    constexpr int AHEAD = 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i <= experts; i += 1024) bins[i] = 0;
    __syncthreads();
    const auto for_slots = [&](const auto &use) {
        for (long long from = tid; from < slots; from += 1024 * AHEAD) {
            int e[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) e[i] = chosen[min(from + 1024 * i, (long long)slots - 1)];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (from + 1024 * i < slots) use((int)(from + 1024 * i), (unsigned)e[i] < (unsigned)experts ? e[i] : experts);
        }
    };
    for_slots([&](int, const int bin) { atomicAdd(&bins[bin], 1); });
    __syncthreads();
    const int each = (experts + 1024) / 1024, first = min(tid * each, experts + 1), last = min(first + each, experts + 1);
    int held = 0, made = 0;  // slots and tiles in front of this thread's bins
    for (int b = first; b < last; ++b) held += bins[b], made += (bins[b] + rows - 1) / rows;
    const int my_held = held, my_made = made;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int a = __shfl_up(held, d), b = __shfl_up(made, d);
        if (lane >= d) held += a, made += b;
    }
    if (lane == 63) sums[0][wave] = held, sums[1][wave] = made;
    __syncthreads();
    for (int w = 0; w < wave; ++w) held += sums[0][w], made += sums[1][w];
    if (tid == 1023) *count = made;
    held -= my_held, made -= my_made;
    for (int b = first; b < last; ++b) {
        const int n = bins[b];
        bins[b] = held;
        for (int i = 0; i < n; i += rows, ++made) *reinterpret_cast<v4i *>(tiles + 4 * (size_t)made) = v4i{b, held + i, min(n - i, rows), 0};
        held += n;
    }
    __syncthreads();
    for_slots([&](const int slot, const int bin) { order[atomicAdd(&bins[bin], 1)] = slot; });
}

// The tile of a workgroup of gemm_grouped_wide_kernel: rows of one expert.
template <int T, int BM, int BN, ExpertsOut OUT>
struct ExpertsTile {
    static constexpr bool PAIRS = OUT == EXPERTS_GATED;
    const ExpertsArgs &p;
    int expert, first, rows, n0;  // n0: in columns of the output
    __device__ __forceinline__ ExpertsTile(const ExpertsArgs &args) : p(args), expert(-1), n0(blockIdx.y * (PAIRS ? BN / 2 : BN))
    {
        if ((int)blockIdx.x >= scalars(p.count)[0]) return;
        const scalar_ints tile = scalars(p.tiles + 4 * (size_t)blockIdx.x);
        expert = tile[0], first = tile[1], rows = tile[2];
    }
    __device__ __forceinline__ bool none() const
    {
        if (expert < 0) return true;
        if (expert < p.experts) return false;
        if constexpr (OUT == EXPERTS_PLAIN) {
            const int columns = min(BN, p.N - n0);
            for (int i = threadIdx.x; i < rows * columns; i += blockDim.x) static_cast<uint16_t *>(p.out)[(size_t)p.order[first + i / columns] * p.N + n0 + i % columns] = 0;
        }
        return true;
    }
    __device__ __forceinline__ const uint16_t *row(const int i) const { return row_of(p, p.order[first + min(i, rows - 1)]); }
    // column j's row of the weights: of 32 columns sixteen gates, then what they gate
    __device__ __forceinline__ size_t weight(const int j) const
    {
        if constexpr (PAIRS) return (size_t)expert * p.N + min(n0 + j / 32 * 16 + j % 16, p.N / 2 - 1) + (j & 16 ? p.N / 2 : 0);
        return (size_t)expert * p.N + min(n0 + j, p.N - 1);
    }
    __device__ __forceinline__ void put(const int i, const int j, const v4f v, const v4f value = {}) const
    {
        const int n = n0 + (PAIRS ? j / 32 * 16 + j % 16 : j), columns = PAIRS ? p.N / 2 : p.N;
        if (n >= columns) return;
        const float bias = OUT == EXPERTS_PLAIN && p.bias != nullptr ? float_of<T>(p.bias[(size_t)expert * p.N + n]) : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + e >= rows) return;
            const size_t at = (size_t)p.order[first + i + e] * columns + n;
            if constexpr (OUT == EXPERTS_PART) static_cast<float *>(p.out)[at] = v[e];
            else if constexpr (OUT == EXPERTS_GATED) static_cast<uint16_t *>(p.out)[at] = round16<T>(gated(v[e], value[e]));
            else static_cast<uint16_t *>(p.out)[at] = round16<T>(p.bias != nullptr ? v[e] + bias : v[e]);
        }
    }
};
template <int T, int BM, int BN>
using ExpertsPlainTile = ExpertsTile<T, BM, BN, EXPERTS_PLAIN>;
template <int T, int BM, int BN>
using ExpertsGatedTile = ExpertsTile<T, BM, BN, EXPERTS_GATED>;
template <int T, int BM, int BN>
using ExpertsPartTile = ExpertsTile<T, BM, BN, EXPERTS_PART>;

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
