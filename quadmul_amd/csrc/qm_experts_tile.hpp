// Many rows to an expert: tiles of rows of one expert times tiles of columns, on v_mfma_f32_32x32x16_f16.
//
// x is made ready once (experts_ready_rows): float16, its elements paired as the nibbles of a dword are, rows without gaps. A bf16 row times a power of two that brings its
// largest element to 2^14 is a float16 row: the eight bits fit, and what falls below float16's normal numbers is off by 2^-39 of the largest element
// at most. So the weights are float16 integers for either type, exact, and nothing is taken off afterwards.
//
// A wave has 32 MT rows and 64 columns and takes 64 of K at a time. x goes straight into the LDS, two steps ahead, the weights' nibbles too, a quad (128 of K) ahead;
// a wave makes floats of its columns' nibbles in registers, seventy instructions for its 8 MT matrix instructions of 32 cycles, so that the LDS holds a quarter of
// what floats would take, and each float is used for 32 MT rows. One barrier a step.
//
// In the LDS a row of x is eight units of sixteen bytes, turned by half the row's number, a quad of a column four, turned by a quarter of the column's: sixteen lanes meet
// every bank once. A product whose tiles are fewer than the CUs has its K in parts, each with sums of its own (EXPERTS_PART), which the kernel that reads them adds in their order.
//
// Bound by nothing alone: 4096 tokens, 2 of 8 experts of 4096 x 11008, float16: the first product 1.67 ms (885 TFLOP/s), the second 0.90 (818); matrix cores busy 50 %, vector
// pipeline 59, and the clock falls to 1.85 GHz; 2.54 ms in all are 1.99 without matrix instructions, 1.83 without loads, 2.39 without the making of floats. 600 tokens,
// 8 of 128 of 2048 x 1024, bf16: 98 and 54 us; vector pipeline busy 60 %, as floats made of a nibble serve 32 rows only, matrix cores 30, memory 2.9 TB/s. us of all of the first with
// other tiles: 128 x 128 2545 to 2611, 128 x 256 of eight waves 2499 (the second product of the 600 tokens slower), 64 x 512 2660, 256 x 128 2680.
#pragma once
#include "qm_experts.hpp"

namespace qm {

typedef float v16f __attribute__((ext_vector_type(16)));

// Tiles of rows that the order goes through the columns with. 4096 tokens, 2 of 8 experts of 4096 x 11008: us with 2, 4, 8, 16 of them 2614, 2540, 2514, 2550; the tiles dealt
// to the XCDs one by one 2694.
constexpr int EXPERTS_BAND = 8;

__host__ __device__ constexpr int ready_stride(const int k) { return (k + 63) / 64 * 64; }
// Rows of x made ready by the waves of a workgroup, `first` the number of the first wave.
struct ExpertsReady {
    const uint16_t *x;
    long long token, choice;  // in elements; `per` rows to a token
    int per, rows, K;
    uint16_t *to;             // [rows, K], K filled up with zeros to a multiple of 64
    float *back;              // [rows]: what sums over a row are multiplied with, negated where an element is no number or infinite; not for float16
};
template <int T>
__device__ __forceinline__ void experts_ready_rows(const ExpertsReady &p, const long long first, const long long waves)
{
    const int lane = threadIdx.x & 63, units = p.K / 8, all = ready_stride(p.K) / 8;
    for (long long row = first; row < p.rows; row += waves) {
        const uint16_t *const x = p.x + row / p.per * p.token + row % p.per * p.choice;
        v4i *const to = reinterpret_cast<v4i *>(p.to + (size_t)row * all * 8);
        if (lane < all - units) to[units + lane] = v4i{};
        if constexpr (T == QM_IN_F16) {
            for (int u = lane; u < units; u += 64) to[u] = paired(*reinterpret_cast<const v4i_half_aligned *>(x + (size_t)u * 8));
        } else {
            uint32_t most = 0, top = 0;  // the exponent of the largest element that is a number, and of the largest
            for (int u = lane; u < units; u += 64) {
                const v4i v = *reinterpret_cast<const v4i_half_aligned *>(x + (size_t)u * 8);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t low = (uint32_t)v[i] >> 7 & 0xFF, high = (uint32_t)v[i] >> 23 & 0xFF;
                    most = max(most, max(low == 255 ? 0 : low, high == 255 ? 0 : high));
                    top = max(top, max(low, high));
                }
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
            const uint32_t up = min(268u - most, 253u);  // 2^14 over the largest, as an exponent; and back
            const float factor = __builtin_bit_cast(float, up << 23);
            const uint32_t lost = __ballot(top == 255) != 0 ? 1 : 0;
            if (lane == 0) p.back[row] = __builtin_bit_cast(float, (254u - up) << 23 | lost << 31);
            for (int u = lane; u < units; u += 64) {
                const v4i v = paired(*reinterpret_cast<const v4i_half_aligned *>(x + (size_t)u * 8));
                v4i out;
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = (int)round16_pair<QM_IN_F16>(__builtin_bit_cast(float, v[i] << 16) * factor, __builtin_bit_cast(float, v[i] & 0xFFFF0000) * factor);
                to[u] = out;
            }
        }
    }
}
// Where element e of a row made ready is.
__device__ __forceinline__ int ready_place(const int e) { return (e & ~7) + ((e & 4) ? 2 * (e & 3) + 1 : 2 * (e & 3)); }

template <int G, int MT, ExpertsOut OUT>
struct ExpertsTileShape {
    static constexpr int WAVES = 4, THREADS = 64 * WAVES, BM = 32 * MT, BN = 64 * WAVES;
    static constexpr int COLUMNS = OUT == EXPERTS_GATED ? BN / 2 : BN;                   // of the output
    static constexpr int X = BM * 128, W = BN * 64, SCALES = 4 / G;                      // bytes of a step and of a quad; scales of a column and quad
    static constexpr int X_LOADS = X / 1024 / WAVES, W_LOADS = W / 1024 / WAVES;         // instructions of a wave
    static constexpr int W_AT = 3 * X, S_AT = W_AT + 2 * W, ROWS_AT = S_AT + WAVES * 2 * SCALES * 256, BYTES = ROWS_AT + BM * 8;
    static __host__ __device__ constexpr int across(const int columns) { return (columns + COLUMNS - 1) / COLUMNS; }
    static_assert(OUT != EXPERTS_GATED || COLUMNS % 64 == 0, "gated products go on to the end of a step of the second product, which wants zeros there");
    static_assert(X_LOADS >= 1 && W_LOADS >= 1, "every wave loads");
    static_assert(BM <= 64, "a lane to a row");
};

template <int T, int S, int G, int MT, ExpertsOut OUT>
__global__ __launch_bounds__(256, 2) void experts_tile_kernel(const ExpertsArgs p)
{
    typedef GroupedWeights<QM_IN_F16> Weights;
    typedef ExpertsTileShape<G, MT, OUT> Shape;
    constexpr bool PAIRS = OUT == EXPERTS_GATED;
    constexpr int SB = S == QM_IN_F32 ? 4 : 2;
    extern __shared__ __align__(16) uint8_t smem[];
    int *const slots = reinterpret_cast<int *>(smem + Shape::ROWS_AT);
    float *const backs = reinterpret_cast<float *>(slots + Shape::BM);
    // An XCD has tiles side by side in an order that goes through the columns with EXPERTS_BAND tiles of rows at a time
    const int columns = PAIRS ? p.N / 2 : p.N, across = Shape::across(columns), there = scalars(p.count)[0], splits = OUT == EXPERTS_PART ? p.splits : 1;
    if ((int)blockIdx.x >= there * across * splits) return;
    const int at = xcd_contiguous_id(blockIdx.x, there * across * splits), split = OUT == EXPERTS_PART ? at / (there * across) : 0, place_in = at - split * there * across, band0 = place_in / (EXPERTS_BAND * across) * EXPERTS_BAND, band = min(EXPERTS_BAND, there - band0), inside = place_in - band0 * across;
    const int block = __builtin_amdgcn_readfirstlane(inside / band), number = __builtin_amdgcn_readfirstlane(band0 + inside - block * band);
    const scalar_ints tile = scalars(p.tiles + 4 * (size_t)number);
    const int expert = tile[0], first = tile[1], rows = tile[2], n0 = block * Shape::COLUMNS;
    const int tid = threadIdx.x;
    if (expert >= p.experts) {
        if constexpr (OUT == EXPERTS_PLAIN) {
            const int some = min(Shape::COLUMNS, columns - n0);
            for (int i = tid; i < rows * some; i += Shape::THREADS) static_cast<uint16_t *>(p.out)[(size_t)p.order[first + i / some] * columns + n0 + i % some] = 0;
        }
        return;
    }
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, h = lane >> 5;
    const int line = p.K / 2, step0 = OUT == EXPERTS_PART ? __builtin_amdgcn_readfirstlane(split) * p.steps_each : 0, steps = OUT == EXPERTS_PART ? min((p.K + 63) / 64, step0 + p.steps_each) : (p.K + 63) / 64;

    for (int i = tid; i < Shape::BM; i += Shape::THREADS) {
        const int slot = p.order[first + min(i, rows - 1)];
        slots[i] = slot;
        backs[i] = p.back != nullptr ? p.back[p.shared ? slot / p.top_k : slot] : 1.0f;
    }
    // ---- where a wave loads from: x, eight lanes to a row of a step; the weights, four to a column's quad; scales, one to a column ----
    // column j of the tile: of a wave's 64 32 are gates, then what they gate
    const auto weight = [&](const int j) {
        if constexpr (PAIRS) return min(n0 + j / 64 * 32 + j % 32, columns - 1) + (j & 32 ? columns : 0);
        else return min(n0 + j, columns - 1);
    };
    const uint8_t *x_at[Shape::X_LOADS];
    uint32_t w_at[Shape::W_LOADS], s_at;
#pragma unroll
    for (int i = 0; i < Shape::X_LOADS; ++i) {
        const int row = (wave * Shape::X_LOADS + i) * 8 + (lane >> 3), slot = p.order[first + min(row, rows - 1)];
        x_at[i] = reinterpret_cast<const uint8_t *>(p.ready + (size_t)(p.shared ? slot / p.top_k : slot) * ready_stride(p.K)) + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int i = 0; i < Shape::W_LOADS; ++i) {
        const int column = (wave * Shape::W_LOADS + i) * 16 + (lane >> 2);
        w_at[i] = (uint32_t)weight(column) * (uint32_t)line + ((lane & 3) ^ ((column >> 2) & 3)) * 16;
    }
    s_at = (uint32_t)weight(wave * 64 + lane) * (uint32_t)(p.groups * SB);
    const uint8_t *const weights = p.B + (size_t)expert * p.N * line, *const scales = static_cast<const uint8_t *>(p.scale) + (size_t)expert * p.N * (p.groups * SB);
    const uint32_t base = (uint32_t)(uintptr_t)smem;
    const uint32_t x_to = __builtin_amdgcn_readfirstlane(base + wave * Shape::X_LOADS * 1024), w_to = __builtin_amdgcn_readfirstlane(base + Shape::W_AT + wave * Shape::W_LOADS * 1024);
    const uint32_t s_to = __builtin_amdgcn_readfirstlane(base + Shape::S_AT + wave * 2 * Shape::SCALES * 256);
    const auto load_x = [&](const int step, const int place) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < Shape::X_LOADS; ++i)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(x_to + place * Shape::X + i * 1024), "v"(x_at[i] + (size_t)step * 128) : "memory", "m0");
    };
    const auto load_w = [&](const int quad) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < Shape::W_LOADS; ++i) {
            // (the last quad may end with the line)
            const int column = (wave * Shape::W_LOADS + i) * 16 + (lane >> 2);
            const uint32_t past = min((uint32_t)quad * 64 + ((lane & 3) ^ ((column >> 2) & 3)) * 16, (uint32_t)line - 16) - ((lane & 3) ^ ((column >> 2) & 3)) * 16;
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(w_to + (quad & 1) * Shape::W + i * 1024), "v"(w_at[i] + past), "s"(weights) : "memory", "m0");
        }
#pragma unroll
        for (int i = 0; i < Shape::SCALES; ++i) {
            const int block = quad * 4 + i * G, group = min(p.magic == 0 ? block : (int)((unsigned long long)block * p.magic >> 32), p.groups - 1);
            const uint8_t *const from = scales + (size_t)group * SB;
            if constexpr (SB == 4) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(s_to + ((quad & 1) * Shape::SCALES + i) * 256), "v"(s_at), "s"(from) : "memory", "m0");
            else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, %2" ::"s"(s_to + ((quad & 1) * Shape::SCALES + i) * 256), "v"(s_at), "s"(from) : "memory", "m0");
        }
    };

    // ---- where it reads: units of x and pieces of a quad come in by exclusive or ----
    const int my_column = wave * 64 + r;
    const uint32_t x_from = r * 128 + ((G == 1 ? 2 * h : 4 * h) ^ ((r >> 1) & 7)) * 16;
    const uint32_t w_from = Shape::W_AT + my_column * 64 + ((G == 1 ? 0 : h) ^ ((my_column >> 2) & 3)) * 16 + (G == 1 ? 8 * h : 0);
    const uint32_t s_from = Shape::S_AT + wave * 2 * Shape::SCALES * 256 + r * 4;

    v16f total[MT][2] = {}, part[MT][2];  // sums of groups times their scales; over the group that is going on
    const auto apply = [&](const int quad, const int i) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t raw = *reinterpret_cast<const uint32_t *>(smem + s_from + ((quad & 1) * Shape::SCALES + i) * 256 + t * 128);
            const float scale = S == QM_IN_F32 ? __builtin_bit_cast(float, raw) : float_of<S == QM_IN_F32 ? QM_IN_F16 : S>((uint16_t)raw);
#pragma unroll
            for (int m = 0; m < MT; ++m) total[m][t] += part[m][t] * scale;
        }
    };
    const auto use = [&](const int step, const int place, auto odd_) __attribute__((always_inline)) {
        constexpr int ODD = decltype(odd_)::value;
        const int quad = step >> 1;
        uint32_t w[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint8_t *const from = smem + (quad & 1) * Shape::W + t * 2048;
            if constexpr (G == 1) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const v2i some = *reinterpret_cast<const v2i *>(from + (w_from ^ (2 * ODD + g) * 16));
                    w[t][2 * g] = (uint32_t)some[0], w[t][2 * g + 1] = (uint32_t)some[1];
                }
            } else {
                const v4i some = *reinterpret_cast<const v4i *>(from + (w_from ^ (2 * ODD) * 16));
#pragma unroll
                for (int i = 0; i < 4; ++i) w[t][i] = (uint32_t)some[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h8 x[MT], f[2];
#pragma unroll
            for (int m = 0; m < MT; ++m) x[m] = *reinterpret_cast<const h8 *>(smem + place * Shape::X + m * 4096 + (x_from ^ (G == 1 ? i / 2 * 4 + i % 2 : i) * 16));
#pragma unroll
            for (int t = 0; t < 2; ++t) f[t] = Weights::of(w[t][i]);
            const bool fresh = G == 1 ? i % 2 == 0 : G == 2 ? i == 0 : i == 0 && !ODD;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int t = 0; t < 2; ++t) part[m][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[m], f[t], fresh ? v16f{} : part[m][t], 0, 0, 0);
            if (G == 1 && i % 2 == 1 && (i == 1 || step * 64 + 32 < p.K)) apply(quad, 2 * ODD + i / 2);
        }
        if (G == 2) apply(quad, ODD);
        if (G == 4 && (ODD || step + 1 == steps)) apply(quad, 0);
    };

    load_x(step0, 0);
    load_w(step0 >> 1);
    if (step0 + 1 < steps) load_x(step0 + 1, 1);
    int place = 0;
    for (int step = step0; step < steps; step += 2) {
        // the step's x, and its quad, have come when no more are on the way than the step before has asked for
        if (step + 2 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(Shape::X_LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int place1 = place == 2 ? 0 : place + 1, place2 = place1 == 2 ? 0 : place1 + 1;
        if (step + 2 < steps) load_x(step + 2, place2), load_w((step >> 1) + 1);
        use(step, place, std::integral_constant<int, 0>{});
        if (step + 1 >= steps) break;
        if (step + 3 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(Shape::X_LOADS + Shape::W_LOADS + Shape::SCALES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (step + 3 < steps) load_x(step + 3, place);
        use(step + 1, place1, std::integral_constant<int, 1>{});
        place = place2;
    }

    // A bf16 row's power of two comes off its sums after the scales: rows far below 2^14 times scales far above 1 can leave float32's range on the way to a result that does not. Where a
    // wave's sums have, it makes them once more, the power of two in front of the scales: by the same instructions, so what was finite keeps its bits, and straight from memory, as it takes
    // scales above 2^88. us without and with this: the MLP of 600 tokens, 8 of 128 of 2048 x 1024, 174.1 and 174.0, of 2048 tokens 383 and 384; a product of 300 tokens, 4 of 32, 2048 x 1024,
    // 25.5 and 25.9. The whole loop over K a second time, on which the workgroup's waves have to agree, cost 2 % of the first and the last.
    const float *last = backs;  // what the sums are multiplied with on their way out
    if constexpr (T != QM_IN_F16) {
        float most[4] = {};  // (NaN if one of them is)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float larger = __builtin_elementwise_maximum(__builtin_fabsf(total[m][0][i]), __builtin_fabsf(total[m][1][i]));
                most[i % 4] = __builtin_elementwise_maximum(most[i % 4], larger);
            }
        const float largest = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most[0], most[1]), __builtin_elementwise_maximum(most[2], most[3]));
        bool over = !(largest < __builtin_inff());
        if (__builtin_expect(__ballot(over) != 0, 0)) {
            // (rows that are not finite themselves stay so, and a padded batch may be full of them: a tenth of 4096 tokens, 2 of 8 of 4096 x 11008, 2697 us, 7216 with those summed again)
            over = false;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    over |= !(__builtin_fabsf(total[m][0][i]) + __builtin_fabsf(total[m][1][i]) < __builtin_inff()) && backs[m * 32 + 8 * (i / 4) + 4 * h + i % 4] > 0.0f;
        }
        if (__builtin_expect(__ballot(over) != 0, 0)) {
            const uint16_t *x_row[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                total[m][0] = total[m][1] = v16f{};
                x_row[m] = p.ready + (size_t)(p.shared ? slots[m * 32 + r] / p.top_k : slots[m * 32 + r]) * ready_stride(p.K);
            }
            for (int step = step0; step < steps; ++step) {
                const int quad = step >> 1, odd = step & 1;
                const auto add = [&](const int i) __attribute__((always_inline)) {
                    const int block = quad * 4 + i * G, group = min(p.magic == 0 ? block : (int)((unsigned long long)block * p.magic >> 32), p.groups - 1);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const float scale = element<S>(scales, (size_t)weight(wave * 64 + 32 * t + r) * p.groups + group);
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int j = 0; j < 16; ++j) total[m][t][j] += part[m][t][j] * __builtin_fabsf(backs[m * 32 + 8 * (j / 4) + 4 * h + j % 4]) * scale;
                    }
                };
                // (pieces of a quad and units of a step as `use` has them; the last quad may end with the line)
                uint32_t w[2][4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t piece = G == 1 ? 2 * odd + i / 2 : h + 2 * odd, dword = G == 1 ? 2 * h + i % 2 : i;
                        const uint32_t from = min((uint32_t)quad * 64 + piece * 16, (uint32_t)line - 16) + dword * 4;
                        w[t][i] = *reinterpret_cast<const uint32_t *>(weights + (size_t)weight(wave * 64 + 32 * t + r) * line + from);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int unit = G == 1 ? 2 * h + i / 2 * 4 + i % 2 : 4 * h + i;
                    const bool fresh = G == 1 ? i % 2 == 0 : i == 0 && (G == 2 || !odd);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const h8 x = *reinterpret_cast<const h8 *>(x_row[m] + (size_t)step * 64 + unit * 8);
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            if (fresh) part[m][t] = v16f{};
                            part[m][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, Weights::of(w[t][i]), part[m][t], 0, 0, 0);
                        }
                    }
                    if (G == 1 && i % 2 == 1 && (i == 1 || step * 64 + 32 < p.K)) add(2 * odd + i / 2);
                }
                if (G == 2) add(odd);
                if (G == 4 && (odd || step + 1 == steps)) add(0);
            }
            // (ones, where this wave's scales were)
            float *const ones = reinterpret_cast<float *>(smem + Shape::S_AT + wave * 2 * Shape::SCALES * 256);
            ones[lane] = 1.0f;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            last = ones;
        }
    }

    // ---- out ----
    const int n = n0 + (PAIRS ? wave * 32 + r : wave * 64 + r);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = m * 32 + 8 * (i / 4) + 4 * h + i % 4;
            if (row >= rows) continue;
            const float back = T == QM_IN_F16 ? 1.0f : __builtin_fabsf(last[row]);
            if constexpr (PAIRS) {
                // (ready for the second product, with zeros to the end of its last step)
                const int stride = p.pairs_out ? ready_stride(columns) : columns;
                const uint16_t out = n < columns ? round16<T>(gated(total[m][0][i] * back, total[m][1][i] * back)) : 0;
                if (n < stride) static_cast<uint16_t *>(p.out)[(size_t)slots[row] * stride + (p.pairs_out ? ready_place(n) : n)] = out;
            } else {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (n + 32 * t >= columns) continue;
                    const float v = total[m][t][i] * back;
                    const size_t to = (size_t)slots[row] * columns + n + 32 * t;
                    if constexpr (OUT == EXPERTS_PART) static_cast<float *>(p.out)[(size_t)split * p.slots * columns + to] = v;
                    else static_cast<uint16_t *>(p.out)[to] = round16<T>(p.bias != nullptr ? v + float_of<T>(p.bias[(size_t)expert * p.N + n + 32 * t]) : v);
                }
            }
        }
}

}  // namespace qm
