// A router's choice: for each token the experts of the highest scores and their weights. The definition is that of include/qm_abi.h.
#pragma once
#include "qm_float16.hpp"

namespace qm {

struct RouteArgs {
    const void *logits;  // [tokens, experts], rows `stride` elements apart
    const float *bias;
    int *chosen;
    float *weights;
    long long stride;
    int tokens, experts, top_k, groups, top_groups;
    int sigmoid, best_two, renormalise;
    int parts;       // lanes to a group of experts, a power of two
    uint32_t magic;  // 2^20 / experts of a group, rounded up: e * magic >> 20 is e's group
    double scale;
};

// The larger a number, the larger its key; NaN like minus infinity, zeros of either sign alike; no number has key 0.
__device__ __forceinline__ uint32_t key_of(const float x)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return x != x ? 0x007FFFFFu : u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(const double x)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
    return x != x ? 0x000FFFFFFFFFFFFFull : u >> 63 ? ~u : u | 1ull << 63;
}

// Over the L lanes (16 or 64, side by side) of a token, the result in all of them: `join` of two values. Lanes turned round inside a row of 16, then rows against rows.
template <int L, class V, class Join>
__device__ __forceinline__ V over_lanes(V v, const Join &join)
{
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(V) / 4)));
    const auto turned = [](const V x, auto by) {
        if constexpr (sizeof(V) == 4) {
            return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + decltype(by)::value, 0xF, 0xF, false));
        } else {
            const Words w = __builtin_bit_cast(Words, x);
            return __builtin_bit_cast(V, (Words{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[0], 0x120 + decltype(by)::value, 0xF, 0xF, false),
                                                (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[1], 0x120 + decltype(by)::value, 0xF, 0xF, false)}));
        }
    };
    v = join(v, turned(v, std::integral_constant<int, 8>{}));
    v = join(v, turned(v, std::integral_constant<int, 4>{}));
    v = join(v, turned(v, std::integral_constant<int, 2>{}));
    v = join(v, turned(v, std::integral_constant<int, 1>{}));
    if constexpr (L == 64) {
        v = join(v, __shfl_xor(v, 16));
        v = join(v, __shfl_xor(v, 32));
    }
    return v;
}

// Bound by its chain of steps for few tokens: one, 6 of 64 experts, 3.5 us, 1.6 of them the launch; 64 tokens, 8 of 256 in 4 of 8 groups, 7.7, most of it exponentials of 64 bits and top_k
// joins over the lanes one after the other; 16384 tokens, 8 of 128, 8.4 MB in 7.6 us (6.8 with the launches overlapped): the same joins, four tokens to a wave.
//
// L lanes to a token, expert number lane + L i in register i of a lane. What is chosen lies next to a border, where 32 bits would decide by
// their rounding: scores are in 64 bits. Without a bias a softmax has the order of its logits (LOGITS): no score is worked out for the choice, and
// with renormalised weights only those of the chosen.
template <int T, int PER, int L, bool LOGITS>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs p)
{
    constexpr int TOKENS = 256 / L;  // of a workgroup
    __shared__ double held[LOGITS ? 1 : TOKENS * PER * L];
    const int lane = threadIdx.x % L, mine = threadIdx.x / L, base = threadIdx.x & 63 & ~(L - 1);
    const double none = -__builtin_inf();
    for (long long token0 = (long long)blockIdx.x * TOKENS; token0 < p.tokens; token0 += (long long)gridDim.x * TOKENS) {
        const bool in = token0 + mine < p.tokens;
        const long long token = in ? token0 + mine : p.tokens - 1;
        const size_t row = (size_t)(token * p.stride);
        float z[PER];
        float most = -__builtin_inff();
        bool nan = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + L * i;
            z[i] = e < p.experts ? element<T>(p.logits, row + e) : -__builtin_inff();
            most = fmaxf(most, z[i]);
            nan |= z[i] != z[i];
        }
        double top = 0.0, total = 1.0;
        if (!p.sigmoid) {
            most = over_lanes<L>(most, [](const float a, const float b) { return fmaxf(a, b); });
            nan = (__ballot(nan) >> base & (L == 64 ? ~0ull : (1ull << L) - 1)) != 0;
            top = most == -__builtin_inff() ? 0.0 : (double)most;
            if (nan || most == __builtin_inff()) top = __builtin_nan("");
        }
        // s of a logit, but for the softmax's sum
        const auto score = [&](const float logit) { return p.sigmoid ? 1.0 / (1.0 + exp(-(double)logit)) : exp((double)logit - top); };
        double s[PER];
        if (!LOGITS || !p.renormalise) {
#pragma unroll
            for (int i = 0; i < PER; ++i) s[i] = lane + L * i < p.experts ? score(z[i]) : 0.0;
            if (!p.sigmoid) {
                total = 0.0;
#pragma unroll
                for (int i = 0; i < PER; ++i) total += s[i];
                total = over_lanes<L>(total, [](const double a, const double b) { return a + b; });
                if (total == 0.0) total = 1.0;
            }
        }
        typedef std::conditional_t<LOGITS, uint32_t, uint64_t> Key;
        Key key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + L * i;
            if constexpr (LOGITS) {
                key[i] = e < p.experts ? key_of(z[i]) : 0;
            } else {
                const double share = s[i] / total, c = p.bias != nullptr ? share + (double)p.bias[min(e, p.experts - 1)] : share;
                // (a softmax without a bias goes by its logits; what a group is worth, by the scores)
                key[i] = e < p.experts ? key_of(p.bias == nullptr && !p.sigmoid ? (double)z[i] : c) : 0;
                held[mine * (PER * L) + e] = c != c ? none : c;
            }
        }
        if constexpr (!LOGITS) {
            if (p.top_groups < p.groups) {
                // `parts` lanes to a group: its largest two scores, then its place among the groups
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const int size = p.experts / p.groups, group = lane / p.parts, sub = lane - group * p.parts;
                double first = none, second = none;
                if (group < p.groups) {
                    for (int i = sub; i < size; i += p.parts) {
                        const double c = held[mine * (PER * L) + group * size + i];
                        second = fmax(second, fmin(first, c));
                        first = fmax(first, c);
                    }
                }
                for (int d = 1; d < p.parts; d *= 2) {
                    const double a = __shfl_xor(first, d), b = __shfl_xor(second, d);
                    second = fmax(fmin(first, a), fmax(second, b));
                    first = fmax(first, a);
                }
                const uint64_t worth = key_of(p.best_two && size > 1 ? first + second : first);
                int place = 0;
                for (int g = 0; g < p.groups; ++g) {
                    const uint64_t other = __shfl(worth, base + g * p.parts);
                    place += other > worth || (other == worth && g < group);
                }
                const uint64_t kept = __ballot(group < p.groups && place < p.top_groups) >> base;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int e = min(lane + L * i, p.experts - 1), g = (int)((uint32_t)e * p.magic >> 20);
                    if (!(kept >> (g * p.parts) & 1)) key[i] = 0;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
        // the largest, top_k times: lane j keeps the j-th
        int kept = 0;
        for (int j = 0; j < p.top_k; ++j) {
            Key best = 0;
            int at = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (key[i] > best) best = key[i], at = lane + L * i;
            if constexpr (LOGITS) {
                const uint64_t both = over_lanes<L>((uint64_t)best << 32 | (uint32_t)~at, [](const uint64_t a, const uint64_t b) { return a > b ? a : b; });
                at = (int)~(uint32_t)both;
            } else {
                const uint64_t largest = over_lanes<L>(best, [](const uint64_t a, const uint64_t b) { return a > b ? a : b; });
                at = (int)over_lanes<L>(best == largest ? (uint32_t)at : 0xFFFFu, [](const uint32_t a, const uint32_t b) { return min(a, b); });
            }
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane + L * i == at) key[i] = 0;
            if (lane == j) kept = at;
        }
        double weight = lane < p.top_k ? score(element<T>(p.logits, row + kept)) : 0.0;
        if (p.renormalise) {
            // (of scores; those of a softmax by their sum, if that is not 0, which divides out)
            const double sum = over_lanes<L>(weight, [](const double a, const double b) { return a + b; });
            weight /= sum == 0.0 ? 1.0 : sum;
        } else {
            weight /= total;
        }
        if (in && lane < p.top_k) {
            p.chosen[token * p.top_k + lane] = kept;
            p.weights[token * p.top_k + lane] = (float)(weight * p.scale);
        }
    }
}

}  // namespace qm
