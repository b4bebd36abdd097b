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
// page), for the weights, each times its value's scale, that are rounded to float16, the type of the second product's operands. A maximum moves only
// when it is passed by 2^8, which leaves the lanes without an exchange in most steps; the largest weight so far is then 2^6 to 2^14 whatever the scales
// of other pages are. float16 has 11 bits down to 2^-14: 2^-20 of the largest at least (2^-28 where it is 2^14), and steps of 2^-24 below: an error of
// at most 2^-31 of the largest, a token. The sum of the weights is of unrounded ones.
#pragma once
#include "qm_kv.hpp"

namespace qm {

struct AttendArgs {
    const uint16_t *q;
    uint16_t *out;
    long long q_token, q_head;
    int heads, causal, window;
    float scale;   // times log2(e)
    int tiles;     // of rows, side by side
    int rows;      // of a tile that are used at most
    int wide;      // not 0: tiles of 64 rows (kv_attend_rows_kernel), so many steps at a time
    // all sequences' steps one after the other cut into as many equal parts (0: a sequence to a workgroup), for each tile and head, and what
    // is left where a sequence is cut: a part's end of one and beginning of another, 16 rows of dim values and their lse each; and the
    // first part of each sequence and their number
    int parts;
    float *part, *lse;
    int2 *cuts;
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

// The steps that rows first .. last (new tokens) have to look at.
struct AttendRange {
    int begin, steps;
};
__device__ __forceinline__ AttendRange attend_range(const KvArgs &c, const AttendArgs &a, const KvSequence &q, const int first, const int last)
{
    const long long most = min((long long)c.width * c.page, 0x7FFFFFFFll - 2 * ATTEND_STEP);
    int end = q.begin + last < 0 || c.pages == 0 || c.width == 0 ? 0 : a.causal ? q.begin + last + 1 : q.length;
    end = (int)min((long long)end, most);
    const int from = a.window > 0 ? max(q.begin + first - a.window + 1, 0) : 0;
    const int begin = from / ATTEND_STEP;
    return {begin, end > from ? (end + ATTEND_STEP - 1) / ATTEND_STEP - begin : 0};
}

// Where part `number` of all sequences' steps begins: in sequence s (-1: past the last one), at the step `at` of it; `per` steps to a part, and
// the sequence's own begin at step number `before`. A wave finds it by itself, a lane to a sequence: the lengths are in device
// memory, and the parts are to be equally long whatever they are.
struct AttendCut {
    int s, per;
    long long before;
};
__device__ __forceinline__ int attend_steps(const KvArgs &c, const AttendArgs &a, const KvSequence &q)
{
    // (a sequence that sees nothing has its rows of zeros: one step)
    return q.count > 0 ? max(attend_range(c, a, q, 0, q.count - 1).steps, 1) : 0;
}
__device__ __forceinline__ AttendCut attend_cut(const KvArgs &c, const AttendArgs &a, const int number)
{
    const int lane = threadIdx.x & 63;
    const auto steps_of = [&](const int s) {
        const int i = min(s, c.sequences - 1), n = c.lengths[i], from = c.start[i], to = c.start[i + c.packed], length = max(n, 0);
        const int lo = c.packed ? min(max(from, 0), c.tokens) : i * c.per, hi = c.packed ? min(max(to, lo), c.tokens) : lo + c.per;
        return s < c.sequences ? attend_steps(c, a, KvSequence{lo, hi - lo, length - (hi - lo), length}) : 0;
    };
    const auto up_to_lane = [&](long long v) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const long long w = __shfl_up(v, d);
            if (lane >= d) v += w;
        }
        return v;
    };
    long long total = 0, up = 0;
    int steps = 0;
    for (int base = 0; base < c.sequences; base += 64) {
        steps = steps_of(base + lane);
        up = up_to_lane(steps);
        total += __shfl(up, 63);
    }
    const int per = (int)min((total + a.parts - 1) / a.parts, 0x7FFFFFFFll);
    const long long from = (long long)number * per;
    long long before = 0;
    for (int base = 0; base < c.sequences; base += 64) {
        if (c.sequences > 64) {
            steps = steps_of(base + lane);
            up = up_to_lane(steps);
        }
        const unsigned long long past = __ballot(before + up > from);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            return {base + at, per, before + __shfl(up - steps, at)};
        }
        before += __shfl(up, 63);
    }
    return {-1, 1, 0};
}

// q^T of one row: float16, bf16 brought into its range by a power of two, with the sign of `scale`. What is left for the scores to be
// multiplied with, 0 or more.
template <int T, int D>
__device__ __forceinline__ float attend_query(const uint16_t *x, const float scale, h8 (&query)[D / 32])
{
    constexpr int J = D / 32;
    const int g = (threadIdx.x & 63) >> 4;
    float v[J][8], most = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int d = j * 32 + 32 <= D / 64 * 64 ? (j / 2) * 64 + 16 * g + 8 * (j & 1) : j * 32 + 8 * g;
        const v4i w = *reinterpret_cast<const v4i_half_aligned *>(x + d);
        if constexpr (T == QM_IN_F16) query[j] = __builtin_bit_cast(h8, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[j][e] = float_of<T>((uint16_t)((uint32_t)w[e / 2] >> (16 * (e & 1))));
            most = fmaxf(most, fabsf(v[j][e]));
        }
    }
    float by = fabsf(scale);
    if constexpr (T != QM_IN_F16) {
        most = across_groups_max(most);
        const int e = max((int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 14, -100);  // the largest becomes 2^14 to 2^15
        const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) query[j][i] = (_Float16)(v[j][i] * down);
        }
        by *= __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
    }
    if (scale < 0.0f) {
#pragma unroll
        for (int j = 0; j < J; ++j) query[j] = -query[j];
    }
    return by;
}

// A row of the softmax so far: the maxima of the scores and of score + log2(scale of the value), the sum.
struct AttendRow {
    float top = ATTEND_LOW, high = ATTEND_LOW, total = 0.0f;
};
// Sixteen scores of a lane (tokens token0 + 4 t + i) into weights for the values: by: what a score is multiplied with, 0 or more; vs: the scale
// of the values; whole: every row sees every token.
template <int DT>
__device__ __forceinline__ void attend_weights(v4f (&score)[4], float by, const float vs, const bool whole, const bool there, const int token0, const int limit,
                                               const int below, AttendRow &row, v4f (&out)[DT], h8 (&weight)[2])
{
    float most = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, score[t][i]);
    }
    most *= by;
    if (!whole) {
        most = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = token0 + 4 * t + i;
                score[t][i] = (there & (j <= limit) & (j > below)) ? score[t][i] * by : -INFINITY;
                most = fmaxf(most, score[t][i]);
            }
        }
        by = 1.0f;
    }
    const float size = vs == 0.0f ? -INFINITY : __builtin_amdgcn_logf(fabsf(vs));
    if (__any(most > row.top + ATTEND_SLACK || most + size > row.high + ATTEND_SLACK)) {
        const float t1 = fmaxf(row.top, across_groups_max(most)), h1 = fmaxf(row.high, across_groups_max(most + size));
        row.total *= __builtin_amdgcn_exp2f(row.top - t1);
        const float shrink = __builtin_amdgcn_exp2f(row.high - h1);
#pragma unroll
        for (int t = 0; t < DT; ++t) out[t] *= shrink;
        row.top = t1, row.high = h1;
    }
    // vs * 2^(top - high + lift): by two factors, for the power alone may leave the float range (the product does only where the
    // weight is below 2^-118 of the largest)
    const float root = __builtin_amdgcn_exp2f(0.5f * fminf(row.top - row.high + ATTEND_LIFT, 126.0f - size));
    // (sixteen tokens that a mask hides count 0 whatever the scale of their page is)
    const float weigh = vs == 0.0f || most == -INFINITY ? 0.0f : vs * root * root;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(score[t][i], by, -row.top));
            row.total += p;
            weight[t / 2][(t & 1) * 4 + i] = (_Float16)(p * weigh);
        }
    }
}
// four channels of each of a lane's tiles of a row; the sum is 0 where nothing is seen
template <int T, int DT>
__device__ __forceinline__ void attend_store(const v4f (&out)[DT], const float sum, const float root, const float by, uint16_t *to)
{
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        const v4f v = sum == 0.0f ? v4f{} : out[t] * root * by;
        *reinterpret_cast<v2i_half_aligned *>(to + 16 * t) = v2i{(int)round16_pair<T>(v[0], v[1]), (int)round16_pair<T>(v[2], v[3])};
    }
}

// blockIdx.x: a head of the cache, and a sequence or (CUT) a part of all sequences; blockIdx.y: a tile of rows. The waves take turns at the steps.
// (Workgroups are dealt to the XCDs in turn: with the heads side by side each has as many long and short sequences as the others.)
// 8 heads of 128 channels: 32 sequences of 1 to 8192 tokens 41 us with the join, 3.4 TB/s; one of 131072 57, 4.7 TB/s; one of 517 9.6, which is its
// chain of loads. Bound by memory where sequences are long, and by the latency of a step otherwise: fewer instructions to make floats of the
// codes (a fifth of all) changed nothing.
template <int T, int D, int NW, bool CUT>
__global__ __launch_bounds__(NW * 64, D > 128 ? 1 : 2) void kv_attend_kernel(const KvArgs c, const AttendArgs a)
{
    constexpr int J = D / 32, DT = D / 16, KW = D / 16;  // products of 32 channels; tiles of 16 channels; words of a lane's part of a key
    constexpr int LD = D + 4;
    __shared__ float joined[NW / 2][16][LD];
    __shared__ float stats[NW][3][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % c.kv_heads, shared = a.heads / c.kv_heads, number = blockIdx.x / c.kv_heads;
    const int page_shift = __builtin_ctz(c.page), page_mask = c.page - 1;

    AttendCut cut{number, 1, 0};
    if constexpr (CUT) {
        cut = attend_cut(c, a, number);
        cut.s = __builtin_amdgcn_readfirstlane(cut.s), cut.per = __builtin_amdgcn_readfirstlane(cut.per);
        if (cut.s < 0) return;
    }
    const long long part_begin = (long long)number * cut.per, part_end = part_begin + cut.per;
    long long before = cut.before;
    for (int s = cut.s; s < c.sequences && (!CUT || before < part_end); s += CUT ? 1 : gridDim.x / c.kv_heads) {
        const KvSequence q = kv_sequence(c, s);
        const int rows = q.count * shared, all_steps = CUT ? attend_steps(c, a, q) : 1;
        const bool begins = !CUT || before >= part_begin, ends = !CUT || before + all_steps <= part_end;
        const int from = begins ? 0 : (int)(part_begin - before), to = ends ? all_steps : (int)(part_end - before);
        if (CUT && begins && rows > 0 && blockIdx.y == 0 && head == 0 && threadIdx.x == 0)
            a.cuts[s] = int2{number, (int)((before + all_steps - 1) / cut.per) - number + 1};
        before += all_steps;
        const int begin0 = CUT ? attend_range(c, a, q, 0, q.count - 1).begin : 0;
        for (int tile = blockIdx.y; tile * 16 < rows; tile += gridDim.y) {
            const int first = tile * 16 / shared, last = min(tile * 16 + 15, rows - 1) / shared;
            const AttendRange range = attend_range(c, a, q, first, last);
            // (a tile that the hint did not promise is done in one piece, by the part that its sequence begins in)
            const bool whole_range = (begins && ends) || tile >= a.tiles || min(rows - tile * 16, 16) > a.rows;
            if (whole_range && !begins) continue;
            const int step0 = whole_range ? range.begin : max(begin0 + from, range.begin);
            const int step1 = whole_range ? range.begin + range.steps : min(begin0 + to, range.begin + range.steps);
            const int row = min(tile * 16 + r, rows - 1), token = row / shared;
            const bool mine = tile * 16 + r < rows;
            const size_t out_row = (size_t)(q.row0 + token) * a.heads + head * shared + row % shared;
            const int position = q.begin + token;
            const int limit = position < 0 ? -1 : a.causal ? position : q.length - 1, below = a.window > 0 ? position - a.window : -1;
            // every row sees tokens sees_from .. sees_to
            const int sees_from = a.window > 0 ? q.begin + last - a.window + 1 : 0;
            const int sees_to = q.begin + first < 0 ? -1 : a.causal ? q.begin + first : q.length - 1;

            h8 query[J];
            const float factor = attend_query<T, D>(a.q + (q.row0 + token) * a.q_token + (long long)(head * shared + row % shared) * a.q_head, a.scale, query);

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
            AttendRow state;
            int step = step0 + wave;
            Pages now{-1, -1}, next{-1, -1};
            if (step < step1) {
                now = pages(step);
                next = pages(min(step + NW, step1 - 1));
                load_keys(step, now);
                load_values(step, now);
#pragma unroll
                for (int j = 0; j < J; ++j) asm volatile("" : "+v"(query[j]));  // waited for here, not in the loop behind the values
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
                const Pages then = pages(min(step + 2 * NW, step1 - 1));  // (in front of the keys: what is waited for last is loaded last)
                if (step + NW < step1) load_keys(step + NW, next);

                const bool whole = step * ATTEND_STEP >= sees_from && step * ATTEND_STEP + ATTEND_STEP - 1 <= sees_to && __all(there);
                h8 weight[2];
                attend_weights(score, by, vs, whole, there, step * ATTEND_STEP + 16 * g, limit, below, state, out, weight);
#pragma unroll
                for (int t = 0; t < DT; ++t) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        out[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(half8_of_codes(values[t][2 * u], values[t][2 * u + 1]), weight[u], out[t], 0, 0, 0);
                }
                if (step + NW < step1) load_values(step + NW, next);
                now = next, next = then;
            }

            // the waves' results into one
            const float top = state.top, high = state.high, total = across_groups_sum(state.total);
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
                if (whole_range) {
                    attend_store<T>(out, sum, root, by, a.out + out_row * D + 4 * g);
                } else {
                    const size_t at = ((size_t)(tile * c.kv_heads + head) * (2 * a.parts) + 2 * number + (begins ? 1 : 0)) * 16 + r;
                    float *const to = a.part + at * D + 4 * g;
#pragma unroll
                    for (int t = 0; t < DT; ++t) *reinterpret_cast<v4f *>(to + 16 * t) = sum == 0.0f ? v4f{} : out[t] * root * by;
                    if (g == 0) a.lse[at] = sum == 0.0f ? -INFINITY : t1 + __builtin_amdgcn_logf(sum);
                }
            }
        }
    }
}

// Many rows of a sequence: 16 to a wave, four waves to 64 tokens. The codes of 64 tokens become float16 once for their four waves, in
// the LDS, in the order that the operands want them; each wave makes a fourth of them from what it loaded while the step before was computed.
// blockIdx.x: a tile of 64 rows, the last ones, which see most, first; blockIdx.y: a head of the cache and a sequence. (The other way
// round each of 8 heads has an XCD, whose CUs read the same lines at the same time: twice as long.) Workgroups are dealt to the 8 XCDs in turn and there
// to 4 parts of an XCD: where the number of tiles is even, the few tiles of sequences with few rows would all be dealt to one or some of the 32. So the first
// tiles are turned by one place from one blockIdx.y to the next, as many of them as the number has powers of two (up to 32). A prompt of 512 tokens
// beside 63 single tokens (32 tiles) 1354 us without, 240 turned among 8, 135 among 32; 16 prompts of 128 on 2000 tokens 120 and 119. Bound by
// what does not run at the same time: of 180 thousand cycles (4 prompts of up to 512 tokens) the vector pipeline is busy 47 %, the LDS 35, the matrix cores 22, and between two
// barriers all waves of a lot multiply, then all make floats. (With 32 rows to a wave and four waves
// 4 prompts of up to 512 tokens took 162 us: the longest sequence had a workgroup to every other CU.)
// LOTS of 64 tokens at a time share the rows: with two the longest sequence's last tiles are done sooner, with one (four workgroups to a CU) fewer waves
// wait for each other. 4 prompts of up to 512 tokens (1024 tiles and heads) 95 us with two, 119 with one; 1 of 4096 (2048) 260 and 265; 8 of 2048
// (8192) 561 and 490 (with the tiles turned, as above, 88, 256 and 459). (With four the registers of 128 channels do not fit: 138 us for the first.)
template <int T, int D, int LOTS>
__global__ __launch_bounds__(256 * LOTS, D > 128 ? 2 : 4) void kv_attend_rows_kernel(const KvArgs c, const AttendArgs a)
{
    constexpr int J = D / 32, DT = D / 16, KW = D / 16, QT = 1, ROWS = 64 * QT, MINE = (DT + 3) / 4;  // MINE: tiles of the values that a wave turns into floats
    struct Floats {
        h8 keys[4][J][64], values[DT][2][64];
    };
    extern __shared__ int8_t in_lds[];
    __shared__ float stats[LOTS][4][QT][3][16];
    const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lot = all_waves >> 2, wave = all_waves & 3, r = lane & 15, g = lane >> 4;
    Floats &lds = reinterpret_cast<Floats *>(in_lds)[lot];
    auto &keys = lds.keys;
    auto &values = lds.values;
    const int head = blockIdx.y % c.kv_heads, shared = a.heads / c.kv_heads;
    const int page_shift = __builtin_ctz(c.page), page_mask = c.page - 1;
    const unsigned apart = min(gridDim.x & -gridDim.x, 32u);  // (a power of two)
    for (int s = blockIdx.y / c.kv_heads; s < c.sequences; s += gridDim.y / c.kv_heads) {
        const KvSequence q = kv_sequence(c, s);
        const int rows = q.count * shared, tiles = (rows + ROWS - 1) / ROWS;
        const unsigned turned = (blockIdx.x & ~(apart - 1)) | ((blockIdx.x + (blockIdx.y * apart >> 5)) & (apart - 1));
        for (int behind = turned; behind < tiles; behind += gridDim.x) {
            const int row0 = (tiles - 1 - behind) * ROWS, last_row = min(row0 + ROWS, rows) - 1;
            const AttendRange range = attend_range(c, a, q, row0 / shared, last_row / shared);
            h8 query[QT][J];
            float factor[QT];
            int limit[QT], below[QT];
            AttendRow state[QT];
            v4f out[QT][DT] = {};
            const int my_row0 = min(row0 + wave * 16 * QT, last_row), my_last = min(my_row0 + 16 * QT - 1, last_row);
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const int row = min(my_row0 + 16 * t + r, last_row), token = row / shared, position = q.begin + token;
                limit[t] = position < 0 ? -1 : a.causal ? position : q.length - 1, below[t] = a.window > 0 ? position - a.window : -1;
                factor[t] = attend_query<T, D>(a.q + (q.row0 + token) * a.q_token + (long long)(head * shared + row % shared) * a.q_head, a.scale, query[t]);
            }
            // tokens that all rows of the wave see, and those that some row may see
            const int first = my_row0 / shared, last = my_last / shared;
            const int sees_from = a.window > 0 ? q.begin + last - a.window + 1 : 0;
            const int sees_to = q.begin + first < 0 ? -1 : a.causal ? q.begin + first : q.length - 1;
            const int may_from = a.window > 0 ? q.begin + first - a.window + 1 : 0, may_to = a.causal ? q.begin + last : q.length - 1;

            // this lane's part of a step: row `wave` of four in the keys, and channels of the values
            uint32_t key_words[KW];
            v4i value_words[MINE];
            const auto key_page = [&](const int step) { return kv_page(c, s, (step * ATTEND_STEP + 16 * (r >> 2)) >> page_shift); };
            const auto value_page = [&](const int step) { return kv_page(c, s, (step * ATTEND_STEP + 16 * g) >> page_shift); };
            float2 scales = {0.0f, 0.0f};
            const auto load = [&](const int step, const int kp, const int vp) {
                const int8_t *const k = c.k + (((size_t)max(kp, 0) * c.kv_heads + head) * c.page + ((step * ATTEND_STEP + 16 * (r >> 2)) & page_mask) + (r & 3) + 4 * wave) * D;
#pragma unroll
                for (int w = 0; w < KW; w += 4) {
                    if (w + 4 <= KW) {
                        const v4i x = *reinterpret_cast<const v4i *>(k + w * 16 + 16 * g);
#pragma unroll
                        for (int e = 0; e < 4; ++e) key_words[w + e] = x[e];
                    } else {
                        const v2i x = *reinterpret_cast<const v2i *>(k + w * 16 + 8 * g);
                        key_words[w] = x[0], key_words[w + 1] = x[1];
                    }
                }
                const size_t at = (size_t)max(vp, 0) * c.kv_heads + head;
                scales = *reinterpret_cast<const float2 *>(c.scales + at * 2);
                const int8_t *const v = c.v + (at * D + r) * c.page + ((step * ATTEND_STEP + 16 * g) & page_mask);
#pragma unroll
                for (int t = 0; t < MINE; ++t)
                    if (DT % 4 == 0 || 4 * t + wave < DT) value_words[t] = *reinterpret_cast<const v4i *>(v + (size_t)(4 * t + wave) * 16 * c.page);
            };
            const auto put_in_place = [&]() {
#pragma unroll
                for (int j = 0; j < J; ++j) keys[wave][j][lane] = half8_of_codes(key_words[2 * j], key_words[2 * j + 1]);
#pragma unroll
                for (int t = 0; t < MINE; ++t) {
                    if (DT % 4 == 0 || 4 * t + wave < DT) {
                        values[4 * t + wave][0][lane] = half8_of_codes((uint32_t)value_words[t][0], (uint32_t)value_words[t][1]);
                        values[4 * t + wave][1][lane] = half8_of_codes((uint32_t)value_words[t][2], (uint32_t)value_words[t][3]);
                    }
                }
            };
            // (all lots go round as often: past its last step one has nothing to compute)
            const int step0 = range.begin + lot, step1 = range.begin + range.steps, turns = (range.steps + LOTS - 1) / LOTS;
            int there_now = -1, kp = -1, vp = -1;
            float2 scales_now = {0.0f, 0.0f};
            if (turns > 0) {
                const int now = min(step0, step1 - 1), next = min(step0 + LOTS, step1 - 1);
                load(now, key_page(now), there_now = value_page(now));
                scales_now = scales;
                kp = key_page(next), vp = value_page(next);
                put_in_place();
            }
            for (int turn = 0; turn < turns; ++turn) {
                __syncthreads();
                const int step = step0 + LOTS * turn;
                const bool there = there_now >= 0;
                const int next = min(step + LOTS, step1 - 1), after = min(step + 2 * LOTS, step1 - 1);
                const int kp2 = key_page(after), vp2 = value_page(after);
                load(next, kp, vp);
                there_now = vp, kp = kp2, vp = vp2;
                const int token0 = step * ATTEND_STEP;
                if (step < step1 && token0 <= may_to && token0 + ATTEND_STEP > may_from) {
                    const bool whole = token0 >= sees_from && token0 + ATTEND_STEP - 1 <= sees_to && __all(there);
                    v4f score[QT][4] = {};
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
#pragma unroll
                        for (int j = 0; j < J; ++j) {
                            const h8 k = keys[t][j][lane];
#pragma unroll
                            for (int n = 0; n < QT; ++n) score[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, query[n][j], score[n][t], 0, 0, 0);
                        }
                    }
                    const float vs = fabsf(scales_now.y) < 0x1p-126f ? 0.0f : scales_now.y;
                    h8 weight[QT][2];
#pragma unroll
                    for (int n = 0; n < QT; ++n)
                        attend_weights(score[n], scales_now.x * factor[n], vs, whole, there, token0 + 16 * g, limit[n], below[n], state[n], out[n], weight[n]);
#pragma unroll
                    for (int t = 0; t < DT; ++t) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const h8 v = values[t][u][lane];
#pragma unroll
                            for (int n = 0; n < QT; ++n) out[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, weight[n][u], out[n][t], 0, 0, 0);
                        }
                    }
                }
                __syncthreads();
                put_in_place();
                scales_now = scales;
            }
            // the other lots' results to the first
            constexpr int PITCH = D + 4, PART = 4 * QT * 16 * PITCH;  // floats of a lot
            static_assert((LOTS - 1) * PART * sizeof(float) <= LOTS * sizeof(Floats));
            float *const joined = reinterpret_cast<float *>(in_lds) + (wave * QT * 16 + r) * PITCH + 4 * g;
            __syncthreads();
            if (lot > 0) {
#pragma unroll
                for (int n = 0; n < QT; ++n) {
                    const float total = across_groups_sum(state[n].total);
                    if (g == 0) stats[lot][wave][n][0][r] = state[n].top, stats[lot][wave][n][1][r] = state[n].high, stats[lot][wave][n][2][r] = total;
#pragma unroll
                    for (int t = 0; t < DT; ++t) *reinterpret_cast<v4f *>(joined + (lot - 1) * PART + n * 16 * PITCH + 16 * t) = out[n][t];
                }
            }
            __syncthreads();
            if (lot == 0) {
#pragma unroll
                for (int n = 0; n < QT; ++n) {
                    const int row = row0 + (wave * QT + n) * 16 + r;
                    float top = state[n].top, high = state[n].high;
#pragma unroll
                    for (int l = 1; l < LOTS; ++l) top = fmaxf(top, stats[l][wave][n][0][r]), high = fmaxf(high, stats[l][wave][n][1][r]);
                    float sum = across_groups_sum(state[n].total) * __builtin_amdgcn_exp2f(state[n].top - top);
                    const float mine = __builtin_amdgcn_exp2f(state[n].high - high);
#pragma unroll
                    for (int t = 0; t < DT; ++t) out[n][t] *= mine;
#pragma unroll
                    for (int l = 1; l < LOTS; ++l) {
                        sum += stats[l][wave][n][2][r] * __builtin_amdgcn_exp2f(stats[l][wave][n][0][r] - top);
                        const float theirs = __builtin_amdgcn_exp2f(stats[l][wave][n][1][r] - high);
#pragma unroll
                        for (int t = 0; t < DT; ++t) out[n][t] += *reinterpret_cast<const v4f *>(joined + (l - 1) * PART + n * 16 * PITCH + 16 * t) * theirs;
                    }
                    const float root = __builtin_amdgcn_exp2f(0.5f * (high - top - ATTEND_LIFT));
                    if (row <= last_row) attend_store<T>(out[n], sum, root, root / sum, a.out + ((size_t)(q.row0 + row / shared) * a.heads + head * shared + row % shared) * D + 4 * g);
                }
            }
            __syncthreads();
        }
    }
}

// The parts of a sequence's rows into one, always in the same order. blockIdx.x: a row of a tile; blockIdx.y: a tile and a head; blockIdx.z: a
// sequence. A part to a wave at a time; bound by the latency of three dependent loads.
template <int T, int D, int NW>
__global__ __launch_bounds__(NW * 64) void kv_join_kernel(const KvArgs c, const AttendArgs a)
{
    constexpr int PER = (D + 63) / 64;
    __shared__ float sums[NW][D], weights[NW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = blockIdx.z, shared = a.heads / c.kv_heads;
    const int2 cut = a.cuts[s];
    const KvSequence q = kv_sequence(c, s);
    const int tile = blockIdx.y / c.kv_heads, head = blockIdx.y % c.kv_heads, row = tile * 16 + blockIdx.x, rows = q.count * shared;
    if (row >= rows || cut.y <= 1 || min(rows - tile * 16, 16) > a.rows) return;
    // part i of the sequence: it begins in the second half of its first one, and goes on in the first halves of the others
    const auto place = [&](const int i) { return ((size_t)blockIdx.y * (2 * a.parts) + 2 * (cut.x + i) + (i == 0 ? 1 : 0)) * 16 + blockIdx.x; };
    float top = -INFINITY;
    for (int i = lane; i < cut.y; i += 64) top = fmaxf(top, a.lse[place(i)]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (top == -INFINITY) top = 0.0f;
    float v[PER] = {}, sum = 0.0f;
#pragma unroll 4
    for (int i = wave; i < cut.y; i += NW) {
        const size_t at = place(i);
        const float w = __builtin_amdgcn_exp2f(a.lse[at] - top);
        sum += w;
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (D % 64 == 0 || lane + 64 * e < D) v[e] += w * a.part[at * D + lane + 64 * e];
    }
    if (lane == 0) weights[wave] = sum;
#pragma unroll
    for (int e = 0; e < PER; ++e)
        if (D % 64 == 0 || lane + 64 * e < D) sums[wave][lane + 64 * e] = v[e];
    __syncthreads();
    if ((int)threadIdx.x < D) {
        const int d = threadIdx.x;
        float all = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) all += weights[w], x += sums[w][d];
        a.out[((size_t)(q.row0 + row / shared) * a.heads + head * shared + row % shared) * D + d] = round16<T>(all == 0.0f ? 0.0f : x / all);
    }
}

// One launch of attention, and one that joins the parts where sequences are cut.
hipError_t launch_attend_f16(const KvArgs &c, const AttendArgs &a, hipStream_t s);
hipError_t launch_attend_bf16(const KvArgs &c, const AttendArgs &a, hipStream_t s);

}  // namespace qm
