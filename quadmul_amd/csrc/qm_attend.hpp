// Attention over the paged 8-bit cache (qm_kv.hpp) on the 16-bit matrix instructions.
//
// One pass over a sequence's tokens with the running maximum and sum of a softmax, 64 tokens to a wave at a time. A row is one new
// token and one of the heads that share a head of the cache; 16 rows make the columns of a tile:
//   scores^T [64 tokens x 16 rows] = K [64 x dim] q^T         four tiles of v_mfma_f32_16x16x32_f16 times dim / 32
//   out^T    [dim x 16 rows]      += V^T [dim x 64] p^T       dim / 16 tiles times two
// An int8 code is a float16 exactly, so the codes go into the products as they are and the scales of their pages outside: the keys' into the
// scores, the values' into the weights p. K is the first operand, row by row as it is stored; the tokens of a 64 are dealt to the rows
// of the four tiles so that the lane that ends up with a score has sixteen consecutive tokens of one row of q, which are at once its part of the
// second operand p^T and the sixteen bytes that it loads of a channel of V. No value crosses a lane between the two products, nothing goes
// through the LDS, and every load is 16 bytes of one page (a page has a multiple of 16 tokens).
//
// Both running maxima are kept in units of log2: `top` of the scores, for the sum, and `high` of score + log2(scale of the value's
// page), for the weights that are rounded to float16: these stay within 2^14 of their largest whatever the scales of other pages
// are (11 bits down to 2^-28 of it). A maximum moves only when it is passed by 2^8, which leaves the lanes without an exchange in most steps.
#pragma once
#include "qm_kv.hpp"

namespace qm {

struct AttendArgs {
    const uint16_t *q;
    uint16_t *out;
    float *part;  // several splits: partial results, splits x rows of dim values, then as many lse, then the splits of each row in use
    long long q_token, q_head;
    int heads, causal, window;
    float scale;      // times log2(e)
    int splits, tiles, per;  // splits of a sequence's steps, tiles of rows side by side, steps of a split (more where the splits are too few)
};

constexpr int ATTEND_STEP = 64;   // tokens
constexpr float ATTEND_LOW = -3e38f;  // below every score: no token seen yet
constexpr float ATTEND_SLACK = 8.0f, ATTEND_LIFT = 6.0f;

// Four int8 to four float16: the byte with its sign bit turned over, under the exponent of 1024, is 1024 + 128 + code.
__device__ __forceinline__ void half_of_codes(const uint32_t w, uint32_t &lo, uint32_t &hi)
{
    const uint32_t x = w ^ 0x80808080u;
    const h2 offset = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) + offset);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) + offset);
}
__device__ __forceinline__ h8 half8_of_codes(const uint32_t a, const uint32_t b)
{
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    uint32_t w0, w1, w2, w3;
    half_of_codes(a, w0, w1);
    half_of_codes(b, w2, w3);
    return __builtin_bit_cast(h8, (u4{w0, w1, w2, w3}));
}
__device__ __forceinline__ float across_groups_max(float v) { v = fmaxf(v, __shfl_xor(v, 16)); return fmaxf(v, __shfl_xor(v, 32)); }
__device__ __forceinline__ float across_groups_sum(float v) { v += __shfl_xor(v, 16); return v + __shfl_xor(v, 32); }

// The steps that a tile of rows first .. last (new tokens) has to look at.
struct AttendRange {
    int begin, steps, per, active;
};
__device__ __forceinline__ AttendRange attend_range(const KvArgs &c, const AttendArgs &a, const KvSequence &q, const int first, const int last)
{
    const long long most = min((long long)c.width * c.page, 0x7FFFFFFFll - 2 * ATTEND_STEP);
    int end = q.begin + last < 0 || c.pages == 0 ? 0 : a.causal ? q.begin + last + 1 : q.length;
    end = (int)min((long long)end, most);
    const int from = a.window > 0 ? max(q.begin + first - a.window + 1, 0) : 0;
    const int begin = from / ATTEND_STEP, steps = end > from ? (end + ATTEND_STEP - 1) / ATTEND_STEP - begin : 0;
    const int per = max(a.per, (steps + a.splits - 1) / a.splits);
    return {begin, steps, per, (steps + per - 1) / per};
}

// blockIdx.x: a split, and a tile of rows; blockIdx.y: a head of the cache; blockIdx.z: a sequence. The waves take turns at the steps of their split.
template <int T, int D, int NW>
__global__ __launch_bounds__(NW * 64, D > 128 ? 1 : 2) void kv_attend_kernel(const KvArgs c, const AttendArgs a)
{
    constexpr int J = D / 32, DT = D / 16, KW = D / 16;  // products of 32 channels; tiles of 16 channels; words of a lane's part of a key
    constexpr int LD = D + 4;
    __shared__ float joined[NW / 2][16][LD];
    __shared__ float stats[NW][3][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int head = blockIdx.y, shared = a.heads / c.kv_heads, split = blockIdx.x % a.splits;
    const int page_shift = __builtin_ctz(c.page), page_mask = c.page - 1;

    for (int s = blockIdx.z; s < c.sequences; s += gridDim.z) {
        const KvSequence q = kv_sequence(c, s);
        const int rows = q.count * shared;
        for (int tile = blockIdx.x / a.splits; tile * 16 < rows; tile += a.tiles) {
            const int first = tile * 16 / shared, last = min(tile * 16 + 15, rows - 1) / shared;
            const AttendRange range = attend_range(c, a, q, first, last);
            if (split > 0 && split >= range.active) continue;
            const int row = min(tile * 16 + r, rows - 1), token = row / shared;
            const bool mine = tile * 16 + r < rows;
            const size_t out_row = (size_t)(q.row0 + token) * a.heads + head * shared + row % shared;
            const int position = q.begin + token;
            const int limit = position < 0 ? -1 : a.causal ? position : q.length - 1, below = a.window > 0 ? position - a.window : -1;
            // every row sees tokens sees_from .. sees_to
            const int sees_from = a.window > 0 ? q.begin + last - a.window + 1 : 0;
            const int sees_to = q.begin + first < 0 ? -1 : a.causal ? q.begin + first : q.length - 1;

            // q^T: float16, bf16 brought into its range by a power of two
            h8 query[J];
            float factor = a.scale;
            {
                const uint16_t *const x = a.q + (q.row0 + token) * a.q_token + (long long)(head * shared + row % shared) * a.q_head;
                float v[J][8], most = 0.0f;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int d = j * 32 + 32 <= D / 64 * 64 ? (j / 2) * 64 + 16 * g + 8 * (j & 1) : j * 32 + 8 * g;
                    const v4i w = mine ? (v4i)*reinterpret_cast<const v4i_half_aligned *>(x + d) : v4i{};
                    if constexpr (T == QM_IN_F16) query[j] = __builtin_bit_cast(h8, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[j][e] = float_of<T>((uint16_t)((uint32_t)w[e / 2] >> (16 * (e & 1))));
                        most = fmaxf(most, fabsf(v[j][e]));
                    }
                }
                if constexpr (T == QM_IN_BF16) {
                    most = across_groups_max(most);
                    const int e = max((int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 14, -100);  // the largest becomes 2^14 to 2^15
                    const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
                    factor *= __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
#pragma unroll
                    for (int j = 0; j < J; ++j) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) query[j][i] = (_Float16)(v[j][i] * down);
                    }
                }
            }

            const int step0 = range.begin + split * range.per, step1 = min(step0 + range.per, range.begin + range.steps);
            struct Pages {
                int key, value;  // of this lane's row of the keys and of its sixteen tokens; -1: none
            };
            const auto pages = [&](const int step) {
                return Pages{kv_page(c, s, (step * ATTEND_STEP + 16 * (r >> 2)) >> page_shift), kv_page(c, s, (step * ATTEND_STEP + 16 * g) >> page_shift)};
            };
            uint32_t keys[4][KW], values[DT][4];
            float key_scale = 0.0f, value_scale = 0.0f;
            const auto load_keys = [&](const int step, const Pages &p) {
                const size_t at = (size_t)max(p.key, 0) * c.kv_heads + head;
                const int8_t *const k = c.k + (at * c.page + ((step * ATTEND_STEP + 16 * (r >> 2)) & page_mask) + (r & 3)) * D;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
#pragma unroll
                    for (int w = 0; w < KW; w += 4) {
                        if (w + 4 <= KW) {
                            const v4i x = *reinterpret_cast<const v4i *>(k + 4 * t * D + w * 16 + 16 * g);
#pragma unroll
                            for (int e = 0; e < 4; ++e) keys[t][w + e] = x[e];
                        } else {
                            const v2i x = *reinterpret_cast<const v2i *>(k + 4 * t * D + w * 16 + 8 * g);
                            keys[t][w] = x[0], keys[t][w + 1] = x[1];
                        }
                    }
                }
                const float2 scales = *reinterpret_cast<const float2 *>(c.scales + ((size_t)max(p.value, 0) * c.kv_heads + head) * 2);
                key_scale = scales.x, value_scale = scales.y;
            };
            const auto load_values = [&](const int step, const Pages &p) {
                const size_t at = (size_t)max(p.value, 0) * c.kv_heads + head;
                const int8_t *const v = c.v + (at * D + r) * c.page + ((step * ATTEND_STEP + 16 * g) & page_mask);
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const v4i x = *reinterpret_cast<const v4i *>(v + (size_t)t * 16 * c.page);
#pragma unroll
                    for (int e = 0; e < 4; ++e) values[t][e] = x[e];
                }
            };

            v4f out[DT] = {};
            float top = ATTEND_LOW, high = ATTEND_LOW, total = 0.0f;
            Pages now{-1, -1}, next{-1, -1};
            int step = step0 + wave;
            if (step < step1) {
                now = pages(step);
                load_keys(step, now);
                load_values(step, now);
                if (step + NW < step1) next = pages(step + NW);
            }
            for (; step < step1; step += NW) {
                v4f score[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    score[t] = v4f{};
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        score[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(half8_of_codes(keys[t][2 * j], keys[t][2 * j + 1]), query[j], score[t], 0, 0, 0);
                }
                const float by = key_scale * factor;
                const float vs = fabsf(value_scale) < 0x1p-126f ? 0.0f : value_scale;
                const bool there = now.value >= 0;
                if (step + NW < step1) load_keys(step + NW, next);

                const int token0 = step * ATTEND_STEP + 16 * g;
                const bool whole = step * ATTEND_STEP >= sees_from && step * ATTEND_STEP + ATTEND_STEP - 1 <= sees_to && __all(there);
                float most = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        score[t][i] *= by;
                        if (!whole) {
                            const int j = token0 + 4 * t + i;
                            if (!(there && j <= limit && j > below)) score[t][i] = -INFINITY;
                        }
                        most = fmaxf(most, score[t][i]);
                    }
                }
                const float size = vs == 0.0f ? -INFINITY : __builtin_amdgcn_logf(fabsf(vs));
                if (__any(most > top + ATTEND_SLACK || most + size > high + ATTEND_SLACK)) {
                    const float t1 = fmaxf(top, across_groups_max(most)), h1 = fmaxf(high, across_groups_max(most + size));
                    total *= __builtin_amdgcn_exp2f(top - t1);
                    const float shrink = __builtin_amdgcn_exp2f(high - h1);
#pragma unroll
                    for (int t = 0; t < DT; ++t) out[t] *= shrink;
                    top = t1, high = h1;
                }
                // vs * 2^(top - high + lift): by two factors, for the power alone may leave the float range (the product does only where the
                // weight is below 2^-118 of the largest)
                const float root = __builtin_amdgcn_exp2f(0.5f * fminf(top - high + ATTEND_LIFT, 126.0f - size));
                const float weigh = vs == 0.0f ? 0.0f : vs * root * root;
                h8 weight[2];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(score[t][i] - top);
                        total += p;
                        // (what a mask hides is 0 whatever the scale of its page is)
                        weight[t / 2][(t & 1) * 4 + i] = (_Float16)(!whole && p == 0.0f ? 0.0f : p * weigh);
                    }
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        out[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(half8_of_codes(values[t][2 * u], values[t][2 * u + 1]), weight[u], out[t], 0, 0, 0);
                }
                if (step + NW < step1) {
                    load_values(step + NW, next);
                    now = next;
                    if (step + 2 * NW < step1) next = pages(step + 2 * NW);
                }
            }

            // the waves' results into one
            total = across_groups_sum(total);
            __syncthreads();
            if (g == 0) stats[wave][0][r] = top, stats[wave][1][r] = high, stats[wave][2][r] = total;
            __syncthreads();
            float t1 = ATTEND_LOW, h1 = ATTEND_LOW, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) t1 = fmaxf(t1, stats[w][0][r]), h1 = fmaxf(h1, stats[w][1][r]);
#pragma unroll
            for (int w = 0; w < NW; ++w) sum += stats[w][2][r] * __builtin_amdgcn_exp2f(stats[w][0][r] - t1);
            const float shrink = __builtin_amdgcn_exp2f(high - h1);
#pragma unroll
            for (int t = 0; t < DT; ++t) out[t] *= shrink;
#pragma unroll
            for (int n = NW / 2; n > 0; n /= 2) {
                if (wave >= n && wave < 2 * n) {
#pragma unroll
                    for (int t = 0; t < DT; ++t) *reinterpret_cast<v4f *>(&joined[wave - n][r][16 * t + 4 * g]) = out[t];
                }
                __syncthreads();
                if (wave < n) {
#pragma unroll
                    for (int t = 0; t < DT; ++t) out[t] += *reinterpret_cast<const v4f *>(&joined[wave][r][16 * t + 4 * g]);
                }
                __syncthreads();
            }
            if (wave == 0 && mine) {
                // (the sum is 0 where nothing is seen)
                const float root = __builtin_amdgcn_exp2f(0.5f * (h1 - t1 - ATTEND_LIFT)), by = root / sum;
                if (a.splits == 1) {
                    uint16_t *const to = a.out + out_row * D + 4 * g;
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
                        const v4f v = sum == 0.0f ? v4f{} : out[t] * root * by;
                        *reinterpret_cast<v2i_half_aligned *>(to + 16 * t) = v2i{(int)round16_pair<T>(v[0], v[1]), (int)round16_pair<T>(v[2], v[3])};
                    }
                } else {
                    const size_t all = (size_t)c.tokens * a.heads;
                    float *const to = a.part + (split * all + out_row) * D + 4 * g;
#pragma unroll
                    for (int t = 0; t < DT; ++t) *reinterpret_cast<v4f *>(to + 16 * t) = sum == 0.0f ? v4f{} : out[t] * root * by;
                    float *const lse = a.part + a.splits * all * D;
                    if (g == 0) lse[split * all + out_row] = sum == 0.0f ? -INFINITY : t1 + __builtin_amdgcn_logf(sum);
                    if (g == 0 && split == 0) reinterpret_cast<int *>(lse + a.splits * all)[out_row] = range.active;
                }
            }
        }
    }
}

// The splits of a row into one: a workgroup to a row, its waves take turns at the splits, always in the same order.
template <int T, int D>
__global__ __launch_bounds__(256) void kv_join_kernel(const float *part, uint16_t *out, const int rows, const int splits)
{
    constexpr int PER = (D + 63) / 64;
    __shared__ float sums[4][D], weights[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float *const lse = part + (size_t)splits * rows * D;
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const int active = min(reinterpret_cast<const int *>(lse + (size_t)splits * rows)[row], splits);
        float top = -INFINITY;
        for (int s = lane; s < active; s += 64) top = fmaxf(top, lse[(size_t)s * rows + row]);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        if (top == -INFINITY) top = 0.0f;
        float v[PER] = {}, sum = 0.0f;
#pragma unroll 4
        for (int s = wave; s < active; s += 4) {
            const float w = __builtin_amdgcn_exp2f(lse[(size_t)s * rows + row] - top);
            const float *const x = part + ((size_t)s * rows + row) * D + lane;
            sum += w;
#pragma unroll
            for (int e = 0; e < PER; ++e)
                if (D % 64 == 0 || lane + 64 * e < D) v[e] += w * x[64 * e];
        }
        __syncthreads();
        if (lane == 0) weights[wave] = sum;
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (D % 64 == 0 || lane + 64 * e < D) sums[wave][lane + 64 * e] = v[e];
        __syncthreads();
        if ((int)threadIdx.x < D) {
            const int d = threadIdx.x;
            const float all = weights[0] + weights[1] + weights[2] + weights[3];
            const float x = sums[0][d] + sums[1][d] + sums[2][d] + sums[3][d];
            out[(size_t)row * D + d] = round16<T>(all == 0.0f ? 0.0f : x / all);
        }
    }
}

// One launch of attention, and one that joins the splits where there are several.
hipError_t launch_attend_f16(const KvArgs &c, const AttendArgs &a, hipStream_t s);
hipError_t launch_attend_bf16(const KvArgs &c, const AttendArgs &a, hipStream_t s);

}  // namespace qm
