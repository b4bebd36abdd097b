// 16-bit activations times the packed int4 weights of each token's experts. Choice j of token t is slot t * top_k + j: its row of x times
// the matrix of its expert. The definitions are those of include/qm_abi.h.
#pragma once
#include "qm_grouped.hpp"

namespace qm {

constexpr int EXPERTS_SORTED = 4096;  // experts at most that the slots are sorted by

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
    uint32_t magic;           // 2^32 / (blocks of a group), rounded up: block * magic >> 32 is the block's group, for a K up to 2^20; 0 for one block
    unsigned long long top_k_magic;  // 2^32 / top_k, rounded up, for less than 2^32 / top_k slots
    // The slots sorted by expert, cut into tiles of rows: their expert, where they begin in `order` and how many they are. After
    // those of the last expert, as number `experts`, slots that have none.
    const int *order, *tiles, *count;  // [slots], [tiles][4]; how many tiles, how many of them of an expert, where the slots without one begin in `order`
};
// How the slots of a call are cut into tiles, and where in the workspace the lists are.
struct ExpertsPlan {
    int rows;   // of a tile; 0: no tiles
    int tiles;  // at most
    size_t order, list, count, bytes;
};
// qm_experts_inst.hip, by the type of x; `few`: x's rows can be loaded sixteen aligned bytes at a time.
hipError_t launch_experts_f16(const ExpertsArgs &p, const ExpertsPlan &plan, int scale_dtype, ExpertsOut out, bool tiled, bool few, hipStream_t s);
hipError_t launch_experts_bf16(const ExpertsArgs &p, const ExpertsPlan &plan, int scale_dtype, ExpertsOut out, bool tiled, bool few, hipStream_t s);

__device__ __forceinline__ const uint16_t *row_of(const ExpertsArgs &p, const int slot)
{
    const int t = slot / p.top_k;
    return p.x + t * p.x_token + (slot - t * p.top_k) * p.x_choice;
}
// silu(gate) * value
__device__ __forceinline__ float gated(const float gate, const float value) { return gate / (1.0f + __expf(-gate)) * value; }

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

// Few rows to an expert. An item is up to R rows of one expert and two tiles of 16 columns (a gate's and its value's where one gates the other); a workgroup goes through a
// run of items, its NW waves each through every NW-th run of 256 of K. A wave loads its runs of the weights (whole lines of 128 bytes), of x and
// of the scales straight into the LDS, the next one as soon as the one before is in registers, on into the next item, and waits for nothing but its own loads: twelve to twenty
// waves of a CU have 80 to 130 KB on the way (two runs of fewer waves were slower: their registers and their LDS cost more waves than that). The waves' sums meet in the LDS, one barrier an item. In the
// LDS the 16 bytes of a line, or of a row of x, are turned round by the number of the line or row, so that no read of sixteen lanes meets a bank twice.
//
// WHOLE: 128 of K have one scale, so a matrix instruction may take its 32 of K from anywhere in them: a lane's sixteen bytes of a column, read as they
// are, are its dwords for four instructions. Else every 32 of K go into sums of their own, and a lane reads its dword of each.
template <bool WHOLE, int R, int NW, ExpertsOut OUT>
struct ExpertsRowsShape {
    static constexpr int C = 2, QUARTERS = (R + 3) / 4;                           // tiles of columns; of 16 rows that have sums
    static constexpr int WEIGHTS = C * 2048, X = R * 512, SCALES = WHOLE ? 1 : 4;  // bytes of a run; instructions
    static constexpr int BIAS = OUT == EXPERTS_PLAIN ? 1 : 0;
    static constexpr int STAGE = WEIGHTS + X + (SCALES + BIAS) * 256;
    static constexpr int RING = NW * STAGE, SUMS = NW * C * QUARTERS * 256, BYTES = RING + 2 * SUMS;
    static constexpr int COLUMNS = OUT == EXPERTS_GATED ? 16 : 32;                  // of the output
    static constexpr int WAVES = NW > 4 || !WHOLE || R > 8 ? 4 : 5;                 // to a SIMD, by the registers
    static constexpr int PER_CU = 163840 / BYTES < WAVES * 4 / NW ? 163840 / BYTES : WAVES * 4 / NW;  // workgroups, by the LDS too
};
template <int T, int S, bool WHOLE, int R, int NW, ExpertsOut OUT>
__global__ __launch_bounds__(64 * NW, (ExpertsRowsShape<WHOLE, R, NW, OUT>::WAVES)) void experts_rows_kernel(const ExpertsArgs p)
{
    typedef GroupedWeights<T> W;
    typedef typename W::frag frag;
    typedef ExpertsRowsShape<WHOLE, R, NW, OUT> Shape;
    constexpr bool PAIRS = OUT == EXPERTS_GATED;
    constexpr int C = Shape::C, COLUMNS = Shape::COLUMNS, SB = S == QM_IN_F32 ? 4 : 2;
    extern __shared__ __align__(16) uint8_t smem[];
    v4f *const sums = reinterpret_cast<v4f *>(smem + Shape::RING);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, c = lane >> 4;
    const int columns = PAIRS ? p.N / 2 : p.N, across = (columns + COLUMNS - 1) / COLUMNS, line = p.K / 2, runs = (line + 127) / 128;

    // ---- this workgroup's items: an equal share of tiles times columns, side by side ----
    const int tiles = scalars(p.count)[1], all = tiles * across, each = all / (int)gridDim.x, rest = all - each * (int)gridDim.x, me = blockIdx.x;
    const int item0 = each * me + min(me, rest), item1 = item0 + each + (me < rest ? 1 : 0);

    // ---- the loading side: where a lane loads from, eight lanes to a line of a column, 32 to a row of x, 32 to the scales of a quad or block ----
    const int line_column = lane >> 3;
    uint32_t w_at[C][2], s_at, b_at, x_at[R / 2];
    const uint8_t *weights, *scales;
    int load_tile = item0 / max(across, 1), load_block = item0 - load_tile * across, load_left = item1 - item0, load_run = wave;
    const auto load_columns = [&] {
        const int n0 = load_block * COLUMNS, last = columns - 1;
        // the row of the weights of column i of tile t
        const auto row = [&](const int t, const int i) { return min(n0 + (PAIRS ? 0 : t * 16) + i, last) + (PAIRS && t ? columns : 0); };
#pragma unroll
        for (int t = 0; t < C; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) w_at[t][h] = (uint32_t)row(t, 8 * h + line_column) * (uint32_t)line;
        const uint32_t mine = (uint32_t)((lane & 16) ? row(1, r) : row(0, r));
        s_at = mine * (uint32_t)(p.groups * SB);
        b_at = mine * 2;
    };
    const auto load_rows = [&] {
        const scalar_ints tile = scalars(p.tiles + 4 * (size_t)load_tile);
        const int expert = tile[0], first = tile[1], rows = tile[2];
        weights = p.B + (size_t)expert * p.N * line;
        scales = static_cast<const uint8_t *>(p.scale) + (size_t)expert * p.N * (p.groups * SB);
        uint32_t at[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint32_t slot = (uint32_t)scalars(p.order)[first + min(i, rows - 1)], t = (uint32_t)(slot * p.top_k_magic >> 32);
            at[i] = (t * (uint32_t)p.x_token + (slot - t * (uint32_t)p.top_k) * (uint32_t)p.x_choice) * 2;
        }
#pragma unroll
        for (int j = 0; j < R / 2; ++j) x_at[j] = at[2 * j] ^ ((at[2 * j] ^ at[2 * j + 1]) & (lane & 32 ? ~0u : 0u));
        load_columns();
        return expert;
    };
    const uint32_t ring = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem + wave * Shape::STAGE);
    int load_expert = 0;
    const auto load_stage = [&]() __attribute__((always_inline)) {
        const uint32_t to = ring;
#pragma unroll
        for (int t = 0; t < C; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t piece = ((lane & 7) ^ (((8 * h + line_column) >> 1) & 7)) * 16, from = w_at[t][h] + min((uint32_t)load_run * 128 + piece, (uint32_t)line - 16);
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to + (2 * t + h) * 1024), "v"(from), "s"(weights) : "memory", "m0");
            }
#pragma unroll
        for (int j = 0; j < R / 2; ++j) {
            const uint32_t piece = ((lane & 31) ^ (2 * j + (lane >> 5))) * 16, from = x_at[j] + min((uint32_t)load_run * 512 + piece, (uint32_t)p.K * 2 - 16);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to + Shape::WEIGHTS + j * 1024), "v"(from), "s"(p.x) : "memory", "m0");
        }
#pragma unroll
        for (int j = 0; j < Shape::SCALES; ++j) {
            // quad lane / 32 of the run, or block 2 j + lane / 32
            const uint32_t block = (uint32_t)load_run * 8 + (WHOLE ? 4 : 1) * (lane >> 5) + 2 * j, group = p.magic == 0 ? block : __umulhi(block, p.magic);
            const uint32_t from = s_at + min(group, (uint32_t)p.groups - 1) * SB;
            if constexpr (SB == 4) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to + Shape::WEIGHTS + Shape::X + j * 256), "v"(from), "s"(scales) : "memory", "m0");
            else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, %2" ::"s"(to + Shape::WEIGHTS + Shape::X + j * 256), "v"(from), "s"(scales) : "memory", "m0");
        }
        if constexpr (Shape::BIAS) {
            // (without a bias: whatever stands first in the scales, which nobody reads)
            const uint8_t *const from = p.bias != nullptr ? reinterpret_cast<const uint8_t *>(p.bias) + (size_t)load_expert * p.N * 2 : scales;
            const uint32_t at = p.bias != nullptr ? b_at : 0;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, %2" ::"s"(to + Shape::WEIGHTS + Shape::X + Shape::SCALES * 256), "v"(at), "s"(from) : "memory", "m0");
        }
    };
    // to this wave's next run
    const auto advance = [&] {
        load_run += NW;
        if (load_run < runs) return;
        load_run = wave;
        if (--load_left == 0) return;
        if (++load_block == across) {
            load_block = 0, ++load_tile;
            load_expert = load_rows();
        } else {
            load_columns();
        }
    };
    const bool works = wave < runs;
    if (item0 < item1 && works) {
        load_expert = load_rows();
        load_stage(), advance();
    }

    // ---- the multiplying side ----
    // (numbers of pieces come into an address by exclusive or: its bits for them are those of the turn)
    const int x_row = min(r, R - 1);
    const uint32_t w_from = (r >> 3) * 1024 + (r & 7) * 128 + (((r >> 1) & 7) ^ (WHOLE ? c : 0)) * 16 + (WHOLE ? 0 : 4 * c);
    const uint32_t x_from = Shape::WEIGHTS + x_row * 512 + (x_row ^ (WHOLE ? 4 * c : c)) * 16;
    int tile = item0 / max(across, 1), block0 = item0 - tile * across, parity = 0;
    int rows = 0, my_slot[(R * COLUMNS + 64 * NW - 1) / (64 * NW)];
    for (int item = item0; item < item1; ++item) {
        if (item == item0 || block0 == across) {
            if (block0 == across) block0 = 0, ++tile;
            const scalar_ints of = scalars(p.tiles + 4 * (size_t)tile);
            const int first = of[1];
            rows = of[2];
            // the slot of the row whose sums a thread puts together
#pragma unroll
            for (int i = 0; i < (int)(sizeof(my_slot) / sizeof(int)); ++i) {
                const int m = ((tid + i * 64 * NW) >> 4) % R;
#pragma unroll
                for (int row = 0; row < R; ++row) {
                    const int slot = scalars(p.order)[first + min(row, rows - 1)];
                    my_slot[i] = m == row ? slot : my_slot[i];
                }
            }
        }
        v4f total[C] = {};
        for (int run = wave; run < runs; run += NW) {
            const uint8_t *const at = smem + wave * Shape::STAGE;
            uint32_t w_here = w_from, x_here = x_from;
            asm("" : "+v"(w_here), "+v"(x_here));  // (sixteen addresses that do not change would take as many registers)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if constexpr (Shape::BIAS) {
                if (run == 0 && p.bias != nullptr) {
#pragma unroll
                    for (int t = 0; t < C; ++t) {
                        const float bias = float_of<T>((uint16_t)*reinterpret_cast<const uint32_t *>(at + Shape::WEIGHTS + Shape::X + Shape::SCALES * 256 + (t * 16 + r) * 4));
                        total[t] = v4f{bias, bias, bias, bias};
                    }
                }
            }
            // 128 of K at a time (all 256 would not leave registers for five waves)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                v4i x[4];
                uint32_t w[C][4], scale[C][WHOLE ? 1 : 4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const v4i *>(at + (x_here ^ (WHOLE ? i : 4 * i) * 16) + q * 256);
#pragma unroll
                for (int t = 0; t < C; ++t) {
                    if constexpr (WHOLE) {
                        const v4i whole = *reinterpret_cast<const v4i *>(at + (w_here ^ q * 64) + t * 2048);
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[t][i] = (uint32_t)whole[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[t][i] = *reinterpret_cast<const uint32_t *>(at + (w_here ^ (4 * q + i) * 16) + t * 2048);
                    }
#pragma unroll
                    for (int i = 0; i < (WHOLE ? 1 : 4); ++i) scale[t][i] = *reinterpret_cast<const uint32_t *>(at + Shape::WEIGHTS + Shape::X + ((WHOLE ? q : 4 * q + i) * 32 + t * 16 + r) * 4);
                }
                // (a 16-bit one is in the lower half of its dword)
                const auto scale_of = [&](const int t, const int i) { return S == QM_IN_F32 ? __builtin_bit_cast(float, scale[t][i]) : float_of<S == QM_IN_F32 ? QM_IN_F16 : S>((uint16_t)scale[t][i]); };
                if (q == 1) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (all of the run is in registers: its place is free)
                    if (load_left > 0) load_stage(), advance();
                }
                const int block = run * 8 + q * 4;  // of 32 of K
                if ((block + 4) * 32 > p.K) {
                    // past the end of K: zeros, which whatever weights and scales meet
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = (block + (WHOLE ? c : i)) * 32 < p.K ? x[i] : v4i{};
                }
                frag xs[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) xs[i] = __builtin_bit_cast(frag, paired(x[i]));
                if constexpr (WHOLE) {
                    v4f start = {}, part[C];
                    if constexpr (W::OFFSET) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) start = W::mfma(xs[i], W::offset(), start);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int t = 0; t < C; ++t) part[t] = W::mfma(xs[i], W::of(w[t][i]), i == 0 ? start : part[t]);
#pragma unroll
                    for (int t = 0; t < C; ++t) total[t] += part[t] * scale_of(t, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v4f start = {};
                        if constexpr (W::OFFSET) start = W::mfma(xs[i], W::offset(), start);
#pragma unroll
                        for (int t = 0; t < C; ++t) total[t] += W::mfma(xs[i], W::of(w[t][i]), start) * scale_of(t, i);
                    }
                }
            }
        }

        // ---- the waves' sums, always in the same order; two places for them, so that one barrier is enough ----
        v4f *const here = sums + parity * (Shape::SUMS / 16);
        parity ^= 1;
#pragma unroll
        for (int t = 0; t < C; ++t)
            if (c < Shape::QUARTERS) here[(wave * C + t) * (Shape::QUARTERS * 16) + lane] = total[t];
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int i = 0; i < (int)(sizeof(my_slot) / sizeof(int)); ++i) {
            const int at = tid + i * 64 * NW, column = at & 15, m = (at >> 4) % R, t = (at >> 4) / R, n = block0 * COLUMNS + t * 16 + column;
            const auto sum = [&](const int of) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) v += here[(w * C + of) * (Shape::QUARTERS * 16) + column + 16 * (m >> 2)][m & 3];
                return v;
            };
            if (at >= R * COLUMNS || m >= rows || n >= columns) continue;
            const size_t to = (size_t)my_slot[i] * columns + n;
            if constexpr (OUT == EXPERTS_PART) static_cast<float *>(p.out)[to] = sum(t);
            else if constexpr (OUT == EXPERTS_GATED) static_cast<uint16_t *>(p.out)[to] = round16<T>(gated(sum(0), sum(1)));
            else static_cast<uint16_t *>(p.out)[to] = round16<T>(sum(t));
        }
        ++block0;
    }

    if constexpr (OUT == EXPERTS_PLAIN) {
        // the slots without an expert: those behind the others
        const int from = scalars(p.count)[2];
        const size_t none = (size_t)(p.slots - from) * p.N;
        for (size_t i = (size_t)blockIdx.x * (64 * NW) + tid; i < none; i += (size_t)gridDim.x * (64 * NW))
            static_cast<uint16_t *>(p.out)[(size_t)p.order[from + i / p.N] * p.N + i % p.N] = 0;
    }
}

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
