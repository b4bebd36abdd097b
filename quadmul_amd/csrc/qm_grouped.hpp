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

// ---- on the matrix cores ------------------------------------------------------------------------------------------------------------
//
// D^T is not formed: x is the first operand of v_mfma_f32_16x16x32_{f16,bf16} and the weights the second, so that a lane ends up with
// four rows of one column n, and the scale of that column's group is one value for the four of them. The weights go in as
// integers and the scale comes after the sum over (a part of) a group: nothing is rounded before the end.
//
// A row of B is cut into blocks of 32 elements, 16 bytes. A lane loads block c of four (c = lane / 16) of its column, and needs the c-th dword
// of each: four instructions that swap registers between rows of lanes turn the one into the other, and then every
// instruction has 32 consecutive k, which lie in one group.
//
// A dword's eight nibbles become pairs (0, 4), (1, 5), (2, 6), (3, 7) of 16-bit floats: u = s + 8 put under an exponent whose last bit is 1. The
// elements of x are paired the same way. float16: 1024 + u (or 1024 + 16 u), less 1032 (times 1/16, less 72): exact. bf16: there is no packed
// arithmetic for it and 128 + u is used as it is; the sum of x times 136 is taken off by one more matrix instruction for each 32 k, which all
// columns share and which goes in front of their own: in float32, where it costs 2^-24 of 136 |sum of 32 x|.
template <int T>
struct GroupedWeights;
template <>
struct GroupedWeights<QM_IN_F16> {
    typedef h8 frag;
    static constexpr bool OFFSET = false;
    static __device__ __forceinline__ frag of(const uint32_t w)
    {
        const uint32_t t = w ^ 0x88888888u, t8 = t >> 8;
        const h2 low = {(_Float16)-1032.0f, (_Float16)-1032.0f}, high = {(_Float16)-72.0f, (_Float16)-72.0f}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
        const auto pair = [](const uint32_t v, const uint32_t mask) { return __builtin_bit_cast(h2, (v & mask) | 0x64006400u); };
        const h2 a = pair(t, 0x000F000Fu) + low, b = pair(t, 0x00F000F0u) * sixteenth + high, c = pair(t8, 0x000F000Fu) + low, d = pair(t8, 0x00F000F0u) * sixteenth + high;
        return frag{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    static __device__ __forceinline__ v4f mfma(const frag a, const frag b, const v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct GroupedWeights<QM_IN_BF16> {
    typedef b8 frag;
    static constexpr bool OFFSET = true;
    static __device__ __forceinline__ frag of(const uint32_t w)
    {
        const uint32_t t = w ^ 0x88888888u;
        const auto pair = [](const uint32_t v) { return (int)((v & 0x000F000Fu) | 0x43004300u); };
        return __builtin_bit_cast(frag, (v4i{pair(t), pair(t >> 4), pair(t >> 8), pair(t >> 12)}));
    }
    static __device__ __forceinline__ frag offset() { return __builtin_bit_cast(frag, (v4i{(int)0xC308C308u, (int)0xC308C308u, (int)0xC308C308u, (int)0xC308C308u})); }  // -136
    static __device__ __forceinline__ v4f mfma(const frag a, const frag b, const v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// eight consecutive elements of x, paired as the nibbles are
__device__ __forceinline__ v4i paired(const v4i x)
{
    const auto low = [](const int a, const int b) { return (int)__builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x05040100u); };
    const auto high = [](const int a, const int b) { return (int)__builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x07060302u); };
    return v4i{low(x[0], x[2]), high(x[0], x[2]), low(x[1], x[3]), high(x[1], x[3])};
}

// lane group c has dwords 0..3 of block c  ->  it has dword c of blocks 0..3
__device__ __forceinline__ void turn_blocks(uint32_t (&w)[4])
{
    const auto swap32 = [](uint32_t &a, uint32_t &b) { const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false); a = r[0], b = r[1]; };
    const auto swap16 = [](uint32_t &a, uint32_t &b) { const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false); a = r[0], b = r[1]; };
    swap32(w[0], w[2]);
    swap32(w[1], w[3]);
    swap16(w[0], w[1]);
    swap16(w[2], w[3]);
}

// How many scales four blocks have: groups of whole 128 (1), of 64 (2), of 32 (4), any other multiple of 32 (0).
constexpr int group_mode(const int group) { return group % 128 == 0 ? 1 : group == 64 ? 2 : group == 32 ? 4 : 0; }

// The scales of four blocks from block `block` on of one column: scale[i] belongs to block + i.
template <int S, int MODE>
__device__ __forceinline__ void load_scales(float (&scale)[4], const void *row, const int block, const int group, const int groups)
{
    if constexpr (MODE == 1) {
        const float s = element<S>(row, (size_t)min(block * 32 / group, groups - 1));
        scale[0] = scale[1] = scale[2] = scale[3] = s;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = MODE == 2 ? (block + i) / 2 : MODE == 4 ? block + i : (block + i) * 32 / group;
            scale[i] = element<S>(row, (size_t)min(at, groups - 1));
        }
    }
}

// Up to 16 MT rows: a workgroup has 16 NT columns, its waves take turns at 256 elements of K (one line of every row of B) and their sums meet in the
// LDS. x comes from the L2, where the workgroups share it. Bound by the weights' way from HBM: two turns of every wave are in
// flight.
template <int T, int S, int MODE, int MT, int NT, int NW>
__global__ __launch_bounds__(NW * 64, 2) void gemm_grouped_skinny_kernel(const GroupedArgs p)
{
    typedef GroupedWeights<T> W;
    typedef typename W::frag frag;
    __shared__ v4f sums[NW][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, c = lane >> 4;
    const int blocks = p.K / 32, turns = (blocks + 7) / 8, n0 = blockIdx.x * 16 * NT;

    const uint8_t *row[NT];
    const uint8_t *scales[NT];
    constexpr int SB = S == QM_IN_F32 ? 4 : 2;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = min(n0 + 16 * t + r, p.N - 1);
        row[t] = p.B + (size_t)n * (p.K / 2);
        scales[t] = static_cast<const uint8_t *>(p.scale) + (size_t)n * p.groups * SB;
    }
    const uint16_t *x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = p.x + min(16 * t + r, p.M - 1) * p.x_stride + 8 * c;

    struct Turn {
        v4i w[NT][2];
        float s[NT][2][4];
    };
    const auto load = [&](Turn &to, const int turn) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                to.w[t][h] = *reinterpret_cast<const v4i *>(row[t] + (size_t)min(turn * 8 + 4 * h + c, blocks - 1) * 16);
                load_scales<S, MODE>(to.s[t][h], scales[t], turn * 8 + 4 * h, p.group, p.groups);
            }
        }
    };
    v4f total[MT][NT] = {};
    const auto use = [&](Turn &in, const int turn) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int block = turn * 8 + 4 * h;
            if (block >= blocks) break;
            v4i xs[MT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int t = 0; t < MT; ++t) xs[t][i] = paired(*reinterpret_cast<const v4i_half_aligned *>(x[t] + (size_t)min(block + i, blocks - 1) * 32));
            }
            uint32_t w[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[t][i] = (uint32_t)in.w[t][h][i];
                turn_blocks(w[t]);
            }
            constexpr int PER = MODE == 1 ? 4 : MODE == 2 ? 2 : 1;  // blocks of one scale
#pragma unroll
            for (int run = 0; run < 4; run += PER) {
                v4f part[MT][NT];
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    v4f begin = {};
                    if constexpr (W::OFFSET) {
#pragma unroll
                        for (int i = run; i < run + PER; ++i)
                            if (block + i < blocks) begin = W::mfma(__builtin_bit_cast(frag, xs[a][i]), W::offset(), begin);
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) part[a][t] = begin;
                }
#pragma unroll
                for (int i = run; i < run + PER; ++i) {
                    if (block + i >= blocks) break;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const frag weights = W::of(w[t][i]);
#pragma unroll
                        for (int a = 0; a < MT; ++a) part[a][t] = W::mfma(__builtin_bit_cast(frag, xs[a][i]), weights, part[a][t]);
                    }
                }
                if (block + run < blocks) {
#pragma unroll
                    for (int a = 0; a < MT; ++a) {
#pragma unroll
                        for (int t = 0; t < NT; ++t) total[a][t] += part[a][t] * in.s[t][h][run];
                    }
                }
            }
        }
    };

    // two turns ahead, in three sets of registers
    Turn one, two, three;
    int turn = wave;
    if (turn < turns) load(one, turn);
    if (turn + NW < turns) load(two, turn + NW);
    while (turn < turns) {
        if (turn + 2 * NW < turns) load(three, turn + 2 * NW);
        use(one, turn);
        turn += NW;
        if (turn >= turns) break;
        if (turn + 2 * NW < turns) load(one, turn + 2 * NW);
        use(two, turn);
        turn += NW;
        if (turn >= turns) break;
        if (turn + 2 * NW < turns) load(two, turn + 2 * NW);
        use(three, turn);
        turn += NW;
    }

#pragma unroll
    for (int a = 0; a < MT; ++a) {
#pragma unroll
        for (int t = 0; t < NT; ++t) sums[wave][a * NT + t][lane] = total[a][t];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < MT * NT * 256; i += NW * 64) {
        const int column = i % (16 * NT), m = i / (16 * NT), n = n0 + column;
        const int at = (m >> 4) * NT + column / 16, from = column % 16 + 16 * ((m & 15) >> 2);
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += sums[w][at][from][m & 3];
        if (m < p.M && n < p.N) p.D[(size_t)m * p.N + n] = round16<T>(p.bias != nullptr ? v + float_of<T>(p.bias[n]) : v);
    }
}

}  // namespace qm
