// 16-bit activations times the packed int4 weights of each token's experts. Choice j of token t is slot t * top_k + j: its row of x times
// the matrix of its expert. The definitions are those of include/qm_abi.h.
#pragma once
#include "qm_grouped.hpp"

namespace qm {

constexpr int EXPERTS_SORTED = 4096;  // experts at most that the slots are sorted by

// What becomes of a slot's products: rounded, with the bias (and zeros where the expert is none of these); the first half of the columns as gates of
// the second, rounded; as they are, to be added up by weight; a token's added up by weight, rounded.
enum ExpertsOut { EXPERTS_PLAIN, EXPERTS_GATED, EXPERTS_PART, EXPERTS_SUM };

struct ExpertsArgs {
    const uint16_t *x;
    long long x_token, x_choice;  // in elements, between tokens and between choices
    const int *chosen;            // [slots]
    const uint8_t *B;             // [experts, N, K/2]
    const void *scale;            // [experts, N, groups]
    const uint16_t *bias;         // [experts, N] or null
    void *out;                    // [slots, N], [slots, N/2] 16-bit, [slots, N] float, or [tokens, N] 16-bit
    const float *shares;          // EXPERTS_SUM: [slots], the weights of the choices
    int slots, top_k, experts, N, K, group, groups;
    // For experts_tile_kernel: x made ready, a row to a token (`shared`) or to a slot, and what a row's sums are multiplied with or null; whether gated products
    // are left ready for the next one.
    const uint16_t *ready;
    const float *back;
    int shared, pairs_out;
    int splits, steps_each;   // EXPERTS_PART: parts of K, each with sums of its own one after the other in `out`, and steps of 64 in each but the last, an even number
    uint32_t magic;           // 2^32 / (blocks of a group), rounded up: block * magic >> 32 is the block's group, for a K up to 2^20; 0 for one block
    unsigned long long top_k_magic;  // 2^32 / top_k, rounded up, for less than 2^32 / top_k slots
    // (null where there are no more than 64 slots, and experts_rows_kernel finds its tiles by itself:) the slots sorted by expert, cut into tiles of rows: their expert, where they begin in `order` and how many they are. After
    // those of the last expert, as number `experts`, slots that have none.
    const int *order, *tiles, *count;  // [slots], [tiles][4]; how many tiles, how many of them of an expert, where the slots without one begin in `order`
};
// How the slots of a call are cut into tiles, and where in the workspace the lists are.
struct ExpertsPlan {
    int rows;   // of a tile; 0: no tiles
    int tiles;  // at most
    size_t order, list, count, bytes;
};
// The kernel for a product: that for any address, the tiles, or that for few rows.
enum ExpertsKernel { EXPERTS_ANY, EXPERTS_TILES, EXPERTS_ROWS };
// qm_experts_inst.hip, by the type of x.
hipError_t launch_experts_f16(const ExpertsArgs &p, const ExpertsPlan &plan, int scale_dtype, ExpertsOut out, ExpertsKernel kernel, hipStream_t s);
hipError_t launch_experts_bf16(const ExpertsArgs &p, const ExpertsPlan &plan, int scale_dtype, ExpertsOut out, ExpertsKernel kernel, hipStream_t s);

__device__ __forceinline__ const uint16_t *row_of(const ExpertsArgs &p, const int slot)
{
    const int t = slot / p.top_k;
    return p.x + t * p.x_token + (slot - t * p.top_k) * p.x_choice;
}
// silu(gate) * value
__device__ __forceinline__ float gated(const float gate, const float value) { return gate / (1.0f + __expf(-gate)) * value; }

// Few rows to an expert. An item is up to R rows of one expert and two tiles of 16 columns (a gate's and its value's where one gates the other); a workgroup goes through a
// run of items, its NW waves each through every NW-th run of 256 of K. A wave loads its runs of the weights (whole lines of 128 bytes), of x and
// of the scales straight into the LDS, the next one as soon as the one before is in registers, on into the next item, and waits for nothing but its own loads: twelve to twenty
// waves of a CU have 100 to 150 KB on the way (two runs of fewer waves were slower: their registers and their LDS cost more waves than that). The waves' sums meet in the LDS. There
// the 16 bytes of a line, or of a row of x, are turned round by the number of the line or row, so that no read of sixteen lanes meets a bank twice.
//
// G: 32 G of K have one scale (G 4, 2 or 1), so a matrix instruction may take its 32 of K from anywhere in them: a lane's 4 G bytes of a column, read as they
// are, are its dwords for G instructions into the same sums.
//
// Bound by memory, and by what lies between a load and the next: 32 tokens, 8 of 128 of 2048 x 1024, bf16: 191 MB in 42 us, 4.5 TB/s, the vector pipeline busy for 67 % of them (it makes floats of
// nibbles), the matrix cores for 26; one token, 2 of 8 of 4096 x 14336: 121 MB in 24 us and 60 in 15. The few wide experts of one token come at 4.9 TB/s, 25 MB of many narrow ones at 2: a wave
// has two to four runs, one after the other's latency.
template <int G, int R, int C, int NW, ExpertsOut OUT>
struct ExpertsRowsShape {
    static constexpr int QUARTERS = (R + 3) / 4;                                   // of 16 rows that have sums
    static constexpr int GROUPS = 8 / G, SCALES = GROUPS * C > 4 ? GROUPS * C / 4 : 1;  // of a run: scales of a column, instructions that load them
    static constexpr int WEIGHTS = C * 2048, X = R * 512, BIAS = OUT == EXPERTS_PLAIN ? 1 : 0;
    static constexpr int STAGE = WEIGHTS + X + (SCALES + BIAS) * 256;               // bytes of a run
    static constexpr int RING = NW * STAGE, SUMS = NW * C * QUARTERS * 256;
    static constexpr int COLUMNS = OUT == EXPERTS_GATED ? C * 8 : C * 16;           // of the output
    static constexpr int WAVES = NW == 16 ? 4 : G == 1 ? (R > 8 ? 3 : 4) : R > 2 * G || NW == 8 ? 4 : 5;  // to a SIMD, by the registers
    static constexpr int of_lds(const int bytes) { return 163840 / bytes < WAVES * 4 / NW ? 163840 / bytes : WAVES * 4 / NW; }
    // Places for the waves' sums: two, for one barrier an item, or one and two barriers where a CU has room for one workgroup more with it: 48 tokens, 6 of 64 of 2048 x 1408 in groups
    // of 64 (R 8), 91.5 us with two, 88.7 with one
    static constexpr int PLACES = of_lds(RING + 2 * SUMS) < of_lds(RING + SUMS) ? 1 : 2;
    static constexpr int BYTES = RING + PLACES * SUMS, PER_CU = of_lds(BYTES);  // workgroups of a CU
};
template <int T, int S, int G, int R, int C, int NW, ExpertsOut OUT>
__global__ __launch_bounds__(64 * NW, (ExpertsRowsShape<G, R, C, NW, OUT>::WAVES)) void experts_rows_kernel(const ExpertsArgs p)
{
    typedef GroupedWeights<T> W;
    typedef typename W::frag frag;
    typedef ExpertsRowsShape<G, R, C, NW, OUT> Shape;
    constexpr bool PAIRS = OUT == EXPERTS_GATED, SUM = OUT == EXPERTS_SUM;
    constexpr int COLUMNS = Shape::COLUMNS, SB = S == QM_IN_F32 ? 4 : 2;
    extern __shared__ __align__(16) uint8_t smem[];
    v4f *const sums = reinterpret_cast<v4f *>(smem + Shape::RING);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, c = lane >> 4;
    const int columns = PAIRS ? p.N / 2 : p.N, across = (columns + COLUMNS - 1) / COLUMNS, line = p.K / 2, runs = (line + 127) / 128;

    // ---- the tiles: of the lists, or, of up to 64 slots, from their experts, a slot to a lane; a token each, with its choices one after the other in K ----
    const bool listed = SUM || p.order != nullptr;
    const int chosen = listed ? 0 : p.chosen[min(lane, p.slots - 1)];
    const uint64_t valid = __ballot(!listed && lane < p.slots && (unsigned)chosen < (unsigned)p.experts);
    // A tile begins with every R-th slot of an expert; its number is that of the tiles that begin in slots before that one. The slots of tile t (and of its expert's tiles
    // behind it), and how many tiles there are in all. A lane finds the slots of its expert bit by bit of the expert's number, whatever experts there are.
    const auto find = [&](const int t, int &expert, uint64_t &of) {
        uint32_t low = (uint32_t)valid, high = (uint32_t)(valid >> 32);
        for (int bits = p.experts - 1, bit = 0; bits >> bit; ++bit) {
            const uint64_t set = __ballot(chosen >> bit & 1);
            const uint32_t flip = (uint32_t)(chosen >> bit & 1) - 1;  // all ones where this lane's bit is not set
            low &= (uint32_t)set ^ flip, high &= (uint32_t)(set >> 32) ^ flip;
        }
        const uint32_t rank = __builtin_amdgcn_mbcnt_hi(high, __builtin_amdgcn_mbcnt_lo(low, 0));
        const uint64_t begins = __ballot((rank & (R - 1)) == 0) & valid;
        const uint64_t here = __ballot(__builtin_amdgcn_mbcnt_hi((uint32_t)(begins >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)begins, 0)) == (uint32_t)t) & begins;
        const int first = __builtin_ctzll(here | 1ull << 63);
        expert = __builtin_amdgcn_readlane(chosen, first);
        of = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)high, first) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)low, first)) >> first << first;
        return (int)__builtin_popcountll(begins);
    };
    // its expert, how many rows it has and their slots (past the last one: that again)
    const auto get_tile = [&](const int t, int &expert, int &rows, int (&slot)[R]) {
        if (p.order != nullptr) {
            const scalar_ints tile = scalars(p.tiles + 4 * (size_t)t);
            const int first = tile[1];
            expert = tile[0], rows = tile[2];
#pragma unroll
            for (int i = 0; i < R; ++i) slot[i] = scalars(p.order)[first + min(i, rows - 1)];
        } else {
            uint64_t of;
            find(t, expert, of);
            rows = min((int)__builtin_popcountll(of), R);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                slot[i] = __builtin_ctzll(of);
                if ((of & (of - 1)) != 0) of &= of - 1;
            }
        }
    };
    int none;
    uint64_t nobody;
    const int tiles = SUM ? p.slots / p.top_k : listed ? scalars(p.count)[1] : find(INT32_MAX, none, nobody), choices = SUM ? p.top_k : 1;

    // ---- this workgroup's items: an equal share of tiles times columns, side by side ----
    const int all = tiles * across, each = all / (int)gridDim.x, rest = all - each * (int)gridDim.x, me = blockIdx.x;
    const int item0 = each * me + min(me, rest), item1 = item0 + each + (me < rest ? 1 : 0);

    // ---- the loading side: where a lane loads from, eight lanes to a line of a column, 32 to a row of x, 32 to the scales of a quad or block ----
    const int line_column = lane >> 3;
    uint32_t w_at[C][2], s_at, b_at, x_at[R / 2];
    const uint8_t *weights, *scales;
    int load_tile = item0 / across, load_block = item0 - load_tile * across, load_left = item1 - item0, load_run = 0, load_choice = 0, load_expert = 0;
    const auto load_columns = [&] {
        const int n0 = load_block * COLUMNS, last = columns - 1;
        // the row of the weights of column i of tile t
        const auto row = [&](const int t, const int i) { return min(n0 + (PAIRS ? 0 : t * 16) + i, last) + (PAIRS && t ? columns : 0); };
#pragma unroll
        for (int t = 0; t < C; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) w_at[t][h] = (uint32_t)row(t, 8 * h + line_column) * (uint32_t)line;
        const uint32_t mine = (uint32_t)(C == 2 && (lane & 16) ? row(1, r) : row(0, r));
        s_at = mine * (uint32_t)(p.groups * SB);
        b_at = mine * 2;
    };
    const auto load_rows = [&] {
        int slot[R], rows = 1;
        if constexpr (SUM) {
#pragma unroll
            for (int i = 0; i < R; ++i) slot[i] = load_tile * p.top_k + load_choice;
            load_expert = scalars(p.chosen)[slot[0]];
            if ((unsigned)load_expert >= (unsigned)p.experts) load_expert = 0;  // (loaded all the same, and not used)
        } else {
            get_tile(load_tile, load_expert, rows, slot);
        }
        weights = p.B + (size_t)load_expert * p.N * line;
        scales = static_cast<const uint8_t *>(p.scale) + (size_t)load_expert * p.N * (p.groups * SB);
        uint32_t at[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint32_t t = (uint32_t)((uint32_t)slot[i] * p.top_k_magic >> 32);
            at[i] = (t * (uint32_t)p.x_token + ((uint32_t)slot[i] - t * (uint32_t)p.top_k) * (uint32_t)p.x_choice) * 2;
        }
#pragma unroll
        for (int j = 0; j < R / 2; ++j) x_at[j] = at[2 * j] ^ ((at[2 * j] ^ at[2 * j + 1]) & (lane & 32 ? ~0u : 0u));
    };
    const uint32_t ring = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem + wave * Shape::STAGE);
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
            // group number `sub` of the run
            const uint32_t sub = (lane / (16 * C) + j * (4 / C)) % Shape::GROUPS, block = (uint32_t)load_run * 8 + sub * G, group = p.magic == 0 ? block : __umulhi(block, p.magic);
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
    // to this wave's next run: `by` further on
    const auto advance = [&](const int by) {
        load_run += by;
        if (load_run < runs) return;
        while (load_run >= runs) load_run -= runs, ++load_choice;
        if (load_choice >= choices) {
            if (--load_left == 0) return;
            load_run = wave, load_choice = 0;
            while (load_run >= runs) load_run -= runs, ++load_choice;
            if (++load_block == across) load_block = 0, ++load_tile;
            if (SUM || load_block == 0) load_rows();
            load_columns();
        } else {
            load_rows();
        }
    };
    const bool works = wave < runs * choices;
    if (item0 < item1 && works) {
        load_run = wave;
        while (load_run >= runs) load_run -= runs, ++load_choice;
        load_rows(), load_columns();
        load_stage(), advance(NW);
    }

    // ---- the multiplying side ----
    // (numbers of pieces come into an address by exclusive or: its bits for them are those of the turn)
    const int x_row = min(r, R - 1);
    const uint32_t w_from = (r >> 3) * 1024 + (r & 7) * 128 + (((r >> 1) & 7) ^ (c * G / 4)) * 16 + c * G % 4 * 4;
    const uint32_t x_from = Shape::WEIGHTS + x_row * 512 + (x_row ^ (c * G)) * 16;
    int tile = item0 / across, block0 = item0 - tile * across, parity = 0, rows = 1;
    size_t to[(R * COLUMNS + 64 * NW - 1) / (64 * NW)];  // where in the output the rows are whose sums a thread puts together
    for (int item = item0; item < item1; ++item) {
        if (item == item0 || block0 == across) {
            if (block0 == across) block0 = 0, ++tile;
            int expert, slot[R];
            if constexpr (!SUM) get_tile(tile, expert, rows, slot);
#pragma unroll
            for (int i = 0; i < (int)(sizeof(to) / sizeof(size_t)); ++i) {
                const int m = ((tid + i * 64 * NW) >> 4) % R;
                int mine = tile;
                if constexpr (!SUM) {
#pragma unroll
                    for (int row = 0; row < R; ++row) mine = m == row ? slot[row] : mine;
                }
                to[i] = (size_t)mine * columns;
            }
        }
        v4f total[C] = {};
        for (int run = wave, choice = 0; works; run += NW) {
            while (run >= runs) run -= runs, ++choice;
            if (choice >= choices) break;
            float share = 1.0f;
            bool counts = true;
            if constexpr (SUM) {
                const int slot = tile * p.top_k + choice;
                counts = (unsigned)scalars(p.chosen)[slot] < (unsigned)p.experts;
                share = __builtin_bit_cast(float, (int)scalars(reinterpret_cast<const int *>(p.shares))[slot]);
            }
            v4f mine[C] = {};  // SUM: of this run, which is one choice's; share times scale may be less than float32 holds, or more
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
                __builtin_amdgcn_sched_barrier(0);
                v4i x[4];
                uint32_t w[C][4], scale[C][4 / G];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const v4i *>(at + (x_here ^ (i / G * 4 * G + i % G) * 16) + q * 256);
#pragma unroll
                for (int t = 0; t < C; ++t) {
#pragma unroll
                    for (int g = 0; g < 4 / G; ++g) {
                        typedef uint32_t Words __attribute__((ext_vector_type(G)));
                        const Words some = *reinterpret_cast<const Words *>(at + (w_here ^ (4 * q + g * G) * 16) + t * 2048);
#pragma unroll
                        for (int i = 0; i < G; ++i) w[t][g * G + i] = some[i];
                        scale[t][g] = *reinterpret_cast<const uint32_t *>(at + Shape::WEIGHTS + Shape::X + ((q * (4 / G) + g) * 16 * C + t * 16 + r) * 4);
                    }
                }
                // (a 16-bit one is in the lower half of its dword)
                const auto scale_of = [&](const int t, const int i) {
                    return S == QM_IN_F32 ? __builtin_bit_cast(float, scale[t][i]) : float_of<S == QM_IN_F32 ? QM_IN_F16 : S>((uint16_t)scale[t][i]);
                };
                if (q == 1) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (all of the run is in registers: its place is free)
                    if (load_left > 0) load_stage(), advance(NW);
                }
                if (!counts) continue;
                const int block = run * 8 + q * 4;  // of 32 of K
                if ((block + 4) * 32 > p.K) {
                    // past the end of K: zeros, whatever weights they meet, and scales of zero, whatever the last one is
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = block * 32 + (i / G * 4 * G + c * G + i % G) * 8 < p.K ? x[i] : v4i{};
#pragma unroll
                    for (int t = 0; t < C; ++t)
#pragma unroll
                        for (int g = 0; g < 4 / G; ++g) scale[t][g] = (block + g * G) * 32 < p.K ? scale[t][g] : 0;
                }
                frag xs[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) xs[i] = __builtin_bit_cast(frag, paired(x[i]));
#pragma unroll
                for (int g = 0; g < 4 / G; ++g) {
                    v4f start = {}, part[C];
                    if constexpr (W::OFFSET) {
#pragma unroll
                        for (int i = 0; i < G; ++i) start = W::mfma(xs[g * G + i], W::offset(), start);
                    }
#pragma unroll
                    for (int i = 0; i < G; ++i)
#pragma unroll
                        for (int t = 0; t < C; ++t) part[t] = W::mfma(xs[g * G + i], W::of(w[t][g * G + i]), i == 0 ? start : part[t]);
#pragma unroll
                    for (int t = 0; t < C; ++t) (SUM ? mine : total)[t] += part[t] * scale_of(t, g);
                }
            }
            if constexpr (SUM) {
                if (counts) {
#pragma unroll
                    for (int t = 0; t < C; ++t) total[t] += mine[t] * share;
                }
            }
        }

        // ---- the waves' sums, always in the same order ----
        v4f *const here = sums + parity * (Shape::SUMS / 16);
        if constexpr (Shape::PLACES == 2) parity ^= 1;
        else if (item > item0) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (those of the item before are read)
#pragma unroll
        for (int t = 0; t < C; ++t)
            if (c < Shape::QUARTERS) here[(wave * C + t) * (Shape::QUARTERS * 16) + lane] = total[t];
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int i = 0; i < (int)(sizeof(to) / sizeof(size_t)); ++i) {
            const int at = tid + i * 64 * NW, column = at & 15, m = (at >> 4) % R, t = (at >> 4) / R, n = block0 * COLUMNS + t * 16 + column;
            const auto sum = [&](const int of) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) v += here[(w * C + of) * (Shape::QUARTERS * 16) + column + 16 * (m >> 2)][m & 3];
                return v;
            };
            if (at >= R * COLUMNS || m >= rows || n >= columns) continue;
            if constexpr (OUT == EXPERTS_PART) static_cast<float *>(p.out)[to[i] + n] = sum(t);
            else if constexpr (OUT == EXPERTS_GATED) static_cast<uint16_t *>(p.out)[to[i] + n] = round16<T>(gated(sum(0), sum(1)));
            else static_cast<uint16_t *>(p.out)[to[i] + n] = round16<T>(sum(t));
        }
        ++block0;
    }

    if constexpr (OUT == EXPERTS_PLAIN) {
        // zeros for the slots without an expert: those behind the others
        const int from = listed ? scalars(p.count)[2] : 0;
        const size_t empty = (size_t)(p.slots - from) * p.N;
        for (size_t i = (size_t)blockIdx.x * (64 * NW) + tid; i < empty; i += (size_t)gridDim.x * (64 * NW)) {
            const size_t slot = listed ? p.order[from + i / p.N] : i / p.N;
            if (listed || !(valid >> slot & 1)) static_cast<uint16_t *>(p.out)[slot * p.N + i % p.N] = 0;
        }
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
                        // Sixteenths of the weights, taken back at the end: eight times a large element, or eight times a large scale, can be more than float32 holds, though the result is not
                        const float lo = (float)((int)((uint32_t)byte << 28) >> 28) * 0.0625f, hi = (float)(byte >> 4) * 0.0625f;
                        v = __builtin_fmaf(__builtin_fmaf(float_of<T>(x[2 * j + 1]), hi, float_of<T>(x[2 * j]) * lo), s, v);
                    }
#pragma unroll
                    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
                    sum[half] = v * 16.0f;
                }
            }
            if (lane != 0) continue;
            if (OUT == EXPERTS_PART) static_cast<float *>(p.out)[slot * p.N + n] = sum[0];
            else if (OUT == EXPERTS_GATED) static_cast<uint16_t *>(p.out)[slot * columns + n] = round16<T>(gated(sum[0], sum[1]));
            else static_cast<uint16_t *>(p.out)[slot * p.N + n] = none ? 0 : round16<T>(p.bias != nullptr ? sum[0] + float_of<T>(p.bias[(size_t)expert * p.N + n]) : sum[0]);
        }
    }
}

// y[t] = sum over a token's choices, in their order, of weight times product; four columns to a thread where N has whole fours. Bound by memory: 4096 tokens, 2 choices of 4096
// columns, 168 MB, 34 us.
template <int T, int V>
__global__ __launch_bounds__(256) void experts_sum_kernel(const float *part, const int splits, const int *chosen, const float *weights, uint16_t *y, const int tokens, const int top_k, const int experts, const int N)
{
    typedef float Values __attribute__((ext_vector_type(V)));
    // (the grid covers the columns; there may be nearly 2^31, and an int does not hold the one behind a grid of them)
    const uint32_t n = blockIdx.x * 256 + threadIdx.x;
    if (n >= (uint32_t)N / V) return;
    for (long long t = blockIdx.y; t < tokens; t += gridDim.y) {
        Values v = {};
        // (the loads of eight choices before the first is used)
        for (int j0 = 0; j0 < top_k; j0 += 8) {
            Values each[8];
            float share[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const size_t slot = (size_t)t * top_k + min(j0 + j, top_k - 1);
                each[j] = *reinterpret_cast<const Values *>(part + slot * N + (size_t)n * V);
                share[j] = weights[slot];
            }
            for (int s = 1; s < splits; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) each[j] += *reinterpret_cast<const Values *>(part + (((size_t)s * tokens + t) * top_k + min(j0 + j, top_k - 1)) * N + (size_t)n * V);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool counts = j0 + j < top_k && (unsigned)chosen[(size_t)t * top_k + min(j0 + j, top_k - 1)] < (unsigned)experts;
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = counts ? __builtin_fmaf(share[j], each[j][e], v[e]) : v[e];
            }
        }
        uint16_t *const to = y + (size_t)t * N + (size_t)n * V;
        if constexpr (V == 4) *reinterpret_cast<v2i_half_aligned *>(to) = v2i{(int)round16_pair<T>(v[0], v[1]), (int)round16_pair<T>(v[2], v[3])};
        else to[0] = round16<T>(v[0]);
    }
}

// A product whose K was cut: y[slot] = the parts' sums in their order, and the bias; zeros where there is no expert.
template <int T, int V>
__global__ __launch_bounds__(256) void experts_join_kernel(const float *part, const int splits, const int *chosen, const uint16_t *bias, uint16_t *y, const int slots, const int experts, const int N)
{
    typedef float Values __attribute__((ext_vector_type(V)));
    const uint32_t n = blockIdx.x * 256 + threadIdx.x;
    if (n >= (uint32_t)N / V) return;
    for (long long slot = blockIdx.y; slot < slots; slot += gridDim.y) {
        const int expert = chosen[slot];
        const bool none = (unsigned)expert >= (unsigned)experts;
        Values v = {};
        if (!none) {
            for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const Values *>(part + ((size_t)s * slots + slot) * N + (size_t)n * V);
            if (bias != nullptr)
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] += float_of<T>(bias[(size_t)expert * N + (size_t)n * V + e]);
        }
        uint16_t *const to = y + (size_t)slot * N + (size_t)n * V;
        if constexpr (V == 4) *reinterpret_cast<v2i_half_aligned *>(to) = v2i{(int)round16_pair<T>(v[0], v[1]), (int)round16_pair<T>(v[2], v[3])};
        else to[0] = round16<T>(v[0]);
    }
}

}  // namespace qm
