// The paged 8-bit cache of keys and values: where things are, storing new tokens, reading pages back. The layout and the rules
// are those of include/qm_abi.h.
#pragma once
#include "qm_float16.hpp"

namespace qm {

struct KvArgs {
    int8_t *k, *v;
    float *scales;
    const int *table, *lengths, *start;
    int pages, kv_heads, page, dim, sequences, width, tokens;
    int per;     // new tokens of every sequence where there is no start
    int packed;  // 1: there is; 0: `start` is `lengths`, so that it can be read all the same
};

// A sequence's new tokens: rows row0 .. row0 + count - 1, of which row0 + i is at position begin + i (padding where that
// is negative); `length` tokens in all.
struct KvSequence {
    int row0, count, begin, length;
};
// Integers that are the same for a whole wave come through the scalar cache: one round trip for the three of them, where vector loads behind
// the test for `start` made three.
typedef const __attribute__((address_space(4))) int *scalar_ints;
__device__ __forceinline__ scalar_ints scalars(const int *p) { return (scalar_ints)(uintptr_t)p; }
__device__ __forceinline__ KvSequence kv_sequence(const KvArgs &c, const int s)
{
    const int n = scalars(c.lengths)[s], from = scalars(c.start)[s], to = scalars(c.start)[s + c.packed];
    const int length = max(n, 0);
    const int lo = c.packed ? min(max(from, 0), c.tokens) : s * c.per;
    const int hi = c.packed ? min(max(to, lo), c.tokens) : lo + c.per;
    return {lo, hi - lo, length - (hi - lo), length};
}
// The page of a sequence's tokens number * page and up, -1 for none. The load is made whatever the number is, at a place inside the table (a
// table without entries has none: the callers have left before): a branch round it would be waited for by itself.
__device__ __forceinline__ int kv_page(const KvArgs &c, const int s, const int number)
{
    const int id = c.table[(size_t)s * c.width + min(number, c.width - 1)];
    return ((number < c.width) & (id >= 0) & (id < c.pages)) ? id : -1;
}

struct KvNewArgs {
    const uint16_t *k, *v, *q;
    uint16_t *q_out;
    long long k_token, k_head, v_token, v_head, q_token, q_head;
    const float *cos, *sin;
    int heads, pairs, positions, interleaved;
};

struct Pair {
    float a, b;
};
// Elements of pair i of a head: those that turn together, and neighbours past them.
__device__ __forceinline__ int2 pair_at(const int i, const int pairs, const int interleaved)
{
    return i < pairs && !interleaved ? int2{i, i + pairs} : int2{2 * i, 2 * i + 1};
}
__device__ __forceinline__ uint32_t magnitude(const float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

// The scale of a page after new values of at most `amax` (both as bit patterns, so that a NaN is the largest), and the factors
// for the new values and for the codes that the page has.
struct PageScale {
    float scale, inverse, ratio;
};
__device__ __forceinline__ PageScale page_scale(const float before, const uint32_t amax)
{
#pragma clang fp contract(off)
    const float mine = __builtin_bit_cast(float, amax) * (1.0f / 127.0f);
    float scale = __builtin_bit_cast(float, max(magnitude(before), magnitude(mine)));
    if (scale < 0x1p-100f) scale = 0.0f;
    // (no code stands for an infinity: times an infinite scale one would be a score of either sign, and the weight of minus infinity is 0)
    if (magnitude(scale) >= 0x7F800000u) scale = __builtin_nanf("");
    return {scale, scale > 0.0f ? 1.0f / scale : 0.0f, scale > 0.0f ? before / scale : 0.0f};
}
__device__ __forceinline__ int code_of(const float scaled) { return (int)fminf(fmaxf(rintf(scaled), -127.0f), 127.0f); }
__device__ __forceinline__ int code_of(const float value, const float factor)
{
#pragma clang fp contract(off)
    return code_of(value * factor);
}

// Sixteen values of a head: eight pairs that turn together (VECTOR: `pairs` is a multiple of eight), or one pair.
template <int T, bool VECTOR>
struct Pairs {
    // HEADS: of the queries, that a thread has at a time, with the same cosines and sines: one 42 us for 4 prompts of up to 2048 tokens in float16 (with
    // reading them back), two 35; four spill. In bf16 the pairs lie in scratch memory with one as with two, 72 bytes a lane: see the kernel
    static constexpr int COUNT = VECTOR ? 8 : 1, HEADS = VECTOR ? 2 : 1;
    Pair v[COUNT];
    int2 at;  // elements of the first pair; with VECTOR the eight a side by side from at.x and the eight b from at.y, or a, b, a, b, .. from at.x
    bool apart;
    __device__ __forceinline__ void place(const int i, const int pairs, const int interleaved)
    {
        at = pair_at(i * COUNT, pairs, interleaved);
        apart = i * COUNT < pairs && !interleaved;
    }
    struct Raw {
        v4i p, q;
    };
    __device__ __forceinline__ Raw get(const uint16_t *x) const
    {
        if constexpr (VECTOR) return {*reinterpret_cast<const v4i_half_aligned *>(x + at.x), *reinterpret_cast<const v4i_half_aligned *>(x + (apart ? at.y : at.x + 8))};
        else return {v4i{x[at.x]}, v4i{x[at.y]}};
    }
    __device__ __forceinline__ void set(const Raw &raw)
    {
        const v4i p = raw.p, q = raw.q;
        const auto half = [](const v4i w, const int e) { return float_of<T>((uint16_t)((uint32_t)w[e / 2] >> (16 * (e & 1)))); };
        if constexpr (VECTOR) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float low = e < 4 ? half(p, 2 * e) : half(q, 2 * e - 8), high = e < 4 ? half(p, 2 * e + 1) : half(q, 2 * e - 7);
                v[e] = apart ? Pair{half(p, e), half(q, e)} : Pair{low, high};
            }
        } else {
            v[0] = Pair{half(p, 0), half(q, 0)};
        }
    }
    // Cosines and sines of lot i at a position.
    struct Angles {
        float c[COUNT], s[COUNT];
        bool turns;
    };
    static __device__ __forceinline__ Angles angles(const KvNewArgs &f, const int position, const int i, const int pairs)
    {
        Angles a{};
        a.turns = i * COUNT < pairs;
        if (!a.turns) return a;
        const bool in = position < f.positions;
        const size_t row = (size_t)(in ? max(position, 0) : 0) * pairs + i * COUNT;
        if constexpr (VECTOR) {
            const auto get = [&](float (&to)[COUNT], const float *from) {
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const v4i w = *reinterpret_cast<const v4i_elem_aligned *>(from + e);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int bits = w[j];
                        to[e + j] = __builtin_bit_cast(float, bits);
                    }
                }
            };
            get(a.c, f.cos + row);
            get(a.s, f.sin + row);
        } else {
            a.c[0] = f.cos[row], a.s[0] = f.sin[row];
        }
#pragma unroll
        for (int e = 0; e < COUNT; ++e) a.c[e] = in ? a.c[e] : __builtin_nanf(""), a.s[e] = in ? a.s[e] : __builtin_nanf("");
        return a;
    }
    // The four products and two sums are rounded one by one: the codes are defined by them.
    __device__ __forceinline__ void turn(const Angles &by)
    {
#pragma clang fp contract(off)
        if (!by.turns) return;
#pragma unroll
        for (int e = 0; e < COUNT; ++e) {
            const float ac = v[e].a * by.c[e], bs = v[e].b * by.s[e], bc = v[e].b * by.c[e], as = v[e].a * by.s[e];
            v[e] = Pair{ac - bs, bc + as};
        }
    }
    __device__ __forceinline__ uint32_t largest() const
    {
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < COUNT; ++e) most = max(most, max(magnitude(v[e].a), magnitude(v[e].b)));
        return most;
    }
    __device__ __forceinline__ void store(uint16_t *out) const
    {
        if constexpr (VECTOR) {
            v4i p, q;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t a = round16_pair<T>(v[2 * e].a, v[2 * e + 1].a), b = round16_pair<T>(v[2 * e].b, v[2 * e + 1].b);
                const uint32_t first = round16_pair<T>(v[e].a, v[e].b), second = round16_pair<T>(v[4 + e].a, v[4 + e].b);
                p[e] = (int)(apart ? a : first), q[e] = (int)(apart ? b : second);
            }
            *reinterpret_cast<v4i_half_aligned *>(out + at.x) = p;
            *reinterpret_cast<v4i_half_aligned *>(out + (apart ? at.y : at.x + 8)) = q;
        } else {
            out[at.x] = round16<T>(v[0].a);
            out[at.y] = round16<T>(v[0].b);
        }
    }
    __device__ __forceinline__ void store_codes(int8_t *to, const float factor) const
    {
        if constexpr (VECTOR) {
            uint32_t p[2] = {}, q[2] = {};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t a = (uint8_t)code_of(v[e].a, factor), b = (uint8_t)code_of(v[e].b, factor);
                if (apart) {
                    p[e / 4] |= a << (8 * (e & 3)), q[e / 4] |= b << (8 * (e & 3));
                } else {
                    (e < 4 ? p : q)[e / 2 % 2] |= a << (16 * (e & 1)) | b << (16 * (e & 1) + 8);
                }
            }
            *reinterpret_cast<v2i_any_aligned *>(to + at.x) = v2i{(int)p[0], (int)p[1]};
            *reinterpret_cast<v2i_any_aligned *>(to + (apart ? at.y : at.x + 8)) = v2i{(int)q[0], (int)q[1]};
        } else {
            to[at.x] = (int8_t)code_of(v[0].a, factor);
            to[at.y] = (int8_t)code_of(v[0].b, factor);
        }
    }
};

// Eight channels of four tokens side by side in a page, as they are in memory: of values, whose codes lie with the tokens of a channel together. Tokens
// outside lo .. hi - 1 are zeros.
template <int T>
struct Square {
    v4i rows[4];
    __device__ __forceinline__ float at(const int t, const int e) const { return float_of<T>((uint16_t)((uint32_t)rows[t][e / 2] >> (16 * (e & 1)))); }
    __device__ __forceinline__ void load(const uint16_t *x, const long long token, const int position, const int lo, const int hi, const int begin)
    {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int p = min(max(position + t, lo), hi - 1);
            rows[t] = *reinterpret_cast<const v4i_half_aligned *>(x + (p - begin) * token);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (position + t < lo || position + t >= hi) rows[t] = v4i{};
    }
    __device__ __forceinline__ uint32_t largest() const
    {
        uint32_t most = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int e = 0; e < 8; ++e) most = max(most, magnitude(at(t, e)));
        }
        return most;
    }
    __device__ __forceinline__ uint32_t codes(const int e, const float factor) const
    {
        uint32_t w = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) w |= (uint32_t)(uint8_t)code_of(at(t, e), factor) << (8 * t);
        return w;
    }
};

// four codes of a page whose scale grows
__device__ __forceinline__ uint32_t recoded(const uint32_t w, const float ratio)
{
    uint32_t out = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) out |= (uint32_t)(uint8_t)code_of((float)(int8_t)(w >> (8 * b)), ratio) << (8 * b);
    return out;
}

// blockIdx.z: a sequence; blockIdx.y: a head and a side (keys, values) of it; blockIdx.x: below `slots` the pages that the
// sequence's new tokens fall into, past it the rotation of its queries. A thread has sixteen or 32 values at a time (its first ones stay in its
// registers between the largest value and the codes; further ones are read again, from the L2). Where a page's codes all change they are put
// together in the LDS and go out in whole lines. 4 prompts of up to 2048 tokens, 2847 in all, 32 heads of queries and 8 of the cache, 66 MB: float16 28 us, 2.3
// TB/s, bound by what 128 registers leave in flight; bf16 41, bound by the scratch memory that the rotation of the queries goes through (without queries both take 21).
template <int T, bool VECTOR>
__global__ __launch_bounds__(256, 4) void kv_append_kernel(const KvArgs c, const KvNewArgs f, const int slots)
{
    extern __shared__ uint32_t image[];  // a page of one head and side
    __shared__ uint32_t largest[4];
    typedef Pairs<T, VECTOR> Lot;
    const int tid = threadIdx.x, lots = c.dim / 2 / Lot::COUNT;  // of a head
    for (int s = blockIdx.z; s < c.sequences; s += gridDim.z) {
        const KvSequence q = kv_sequence(c, s);
        if ((int)blockIdx.x >= slots) {
            // a lot of HEADS heads of a token, tokens in turn
            const int each = (f.heads + Lot::HEADS - 1) / Lot::HEADS * lots, across = min(each, 256), stride = (int)(gridDim.x - slots) * gridDim.y * (256 / across);
            if (tid >= 256 / across * across) continue;
            for (int t = ((int)(blockIdx.x - slots) * gridDim.y + blockIdx.y) * (256 / across) + tid / across; t < q.count; t += stride) {
                const int position = q.begin + t;
                for (int i = tid % across; i < each; i += across) {
                    const int head0 = i / lots * Lot::HEADS, lot = i % lots;
                    Lot v;
                    v.place(lot, f.pairs, f.interleaved);
                    typename Lot::Raw raw[Lot::HEADS];
#pragma unroll
                    for (int h = 0; h < Lot::HEADS; ++h) raw[h] = v.get(f.q + (q.row0 + t) * f.q_token + min(head0 + h, f.heads - 1) * f.q_head);
                    const typename Lot::Angles by = Lot::angles(f, position, lot, f.pairs);
#pragma unroll
                    for (int h = 0; h < Lot::HEADS; ++h) {
                        v.set(raw[h]);
                        v.turn(by);
                        if (position < 0) {
#pragma unroll
                            for (int e = 0; e < Lot::COUNT; ++e) v.v[e] = Pair{0.0f, 0.0f};
                        }
                        if (head0 + h < f.heads) v.store(f.q_out + ((size_t)(q.row0 + t) * f.heads + head0 + h) * c.dim);
                    }
                }
            }
            continue;
        }
        const int head = blockIdx.y >> 1, side = blockIdx.y & 1, first = max(q.begin, 0);
        if (q.count == 0 || q.length <= first || c.width == 0) continue;
        const uint16_t *const x = (side ? f.v + head * f.v_head : f.k + head * f.k_head) + q.row0 * (side ? f.v_token : f.k_token);
        const int last = min((q.length - 1) / c.page, c.width - 1), fours = c.page / 4, words = c.page * c.dim / 4;
        for (int number = first / c.page + blockIdx.x; number <= last; number += slots) {
            const int id = kv_page(c, s, number);
            if (id < 0) continue;
            const int base = number * c.page, lo = max(first, base), hi = min(q.length - base, c.page) + base;
            float *const held = c.scales + ((size_t)id * c.kv_heads + head) * 2 + side;
            const float before = lo > base ? *held : 0.0f;
            uint32_t *const codes = reinterpret_cast<uint32_t *>((side ? c.v : c.k) + ((size_t)id * c.kv_heads + head) * c.page * c.dim);
            // keys: a lot of a token; values: eight channels of four tokens. `word` of a page's image in the LDS: the values' have
            // their places in a channel's row turned over by the number of the eight, so that squares side by side meet no bank twice.
            const int squares = c.dim / 8, four0 = (lo - base) / 4, all = side ? ((hi - base + 3) / 4 - four0) * squares : (hi - lo) * lots;
            const auto channel = [&](const int i) { return i % squares * 8; };
            const auto four = [&](const int i) { return four0 + i / squares; };
            const auto word = [&](const int d, const int t4) { return d * fours + (t4 ^ (d / 8 & (fours - 1))); };
            const auto key = [&](Lot &v, const int i) {
                const int t = i / lots, lot = i - t * lots;
                v.place(lot, f.pairs, f.interleaved);
                v.set(v.get(x + (lo + t - q.begin) * f.k_token));
                v.turn(Lot::angles(f, lo + t, lot, f.pairs));
            };
            const auto square = [&](Square<T> &v, const int i) { v.load(x + channel(i), f.v_token, base + 4 * four(i), lo, hi, q.begin); };
            const auto put_key = [&](const Lot &v, const int i, const float inverse, const bool whole) { v.store_codes(reinterpret_cast<int8_t *>(whole ? image : codes) + (lo - base + i / lots) * c.dim, inverse); };
            const auto put_square = [&](const Square<T> &v, const int i, const float inverse, const bool whole) {
                const int d = channel(i), t4 = four(i);
                uint32_t mine = 0;  // the bytes of the new tokens
#pragma unroll
                for (int t = 0; t < 4; ++t) mine |= base + 4 * t4 + t >= lo && base + 4 * t4 + t < hi ? 0xFFu << (8 * t) : 0u;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uint32_t *const at = whole ? image + word(d + e, t4) : codes + (d + e) * fours + t4;
                    const uint32_t w = v.codes(e, inverse);
                    *at = mine == ~0u ? w : (*at & ~mine) | (w & mine);  // (no other thread has this word)
                }
            };
            // (one of the two below is run: as one body, so that neither has registers of the other)
            const auto run = [&](auto first_of, const auto &get, const auto &put_codes) {
                uint32_t amax = 0;
                if (tid < all) {
                    get(first_of, tid);
                    amax = first_of.largest();
                }
                for (int i = tid + 256; i < all; i += 256) {
                    auto v = first_of;
                    get(v, i);
                    amax = max(amax, v.largest());
                }
#pragma unroll
                for (int d = 32; d > 0; d >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
                __syncthreads();  // (the page before is done with)
                if ((tid & 63) == 0) largest[tid >> 6] = amax;
                __syncthreads();
                amax = max(max(largest[0], largest[1]), max(largest[2], largest[3]));

                const PageScale to = page_scale(before, amax);
                const bool whole = lo == base || magnitude(to.scale) != magnitude(before);
                if (whole) {
                    for (int i = tid; i < words; i += 256) {
                        const int at = side ? word(i / fours, i % fours) : i;
                        image[at] = lo > base ? recoded(codes[i], to.ratio) : 0;
                    }
                    __syncthreads();  // (and every thread has read the scale)
                    if (tid == 0) *held = to.scale;
                }
                if (tid < all) put_codes(first_of, tid, to.inverse, whole);
                for (int i = tid + 256; i < all; i += 256) {
                    auto v = first_of;
                    get(v, i);
                    put_codes(v, i, to.inverse, whole);
                }
                if (whole) {
                    __syncthreads();
                    for (int i = tid * 4; i < words; i += 256 * 4) {
                        v4i w;
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = (int)image[side ? word(i / fours, i % fours + e) : i + e];
                        *reinterpret_cast<v4i *>(codes + i) = w;
                    }
                }
            };
            if (side) run(Square<T>{}, square, put_square);
            else run(Lot{}, key, put_key);
        }
    }
}

// The same for few new tokens to a sequence: a wave to a page, a head and a side of it, or to a token's head of the queries, a lane to a pair or a
// channel. No barrier and no LDS: a word that has new codes is put together by the lane that stores them, every other one of a page that
// begins anew or is rounded again by another. Values are read twice, the second time from the cache. Bound by latency: lengths, table, values, and
// the rounding of a page whose scale grows, dword after dword by one wave. 64 sequences, 8 heads of 128, a token each in a graph: 4.9 us where no scale
// grows; a token after the other from the first to the last of a page, mean 7.7 in pages of 16 tokens, 30 in pages of 128 (one head of 256: 37).
template <int T>
__global__ __launch_bounds__(256) void kv_append_few_kernel(const KvArgs c, const KvNewArgs f, const int slots, const int tasks)
{
    typedef Pairs<T, false> Lot;
    const int lane = threadIdx.x & 63, task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), half = c.dim / 2;
    if (task >= tasks) return;
    for (int s = blockIdx.y; s < c.sequences; s += gridDim.y) {
        const KvSequence q = kv_sequence(c, s);
        if (task >= slots * 2 * c.kv_heads) {
            const int heads = tasks - slots * 2 * c.kv_heads;  // (a multiple of the queries' heads)
            for (int i = task - slots * 2 * c.kv_heads; i < q.count * f.heads; i += heads) {
                const int t = i / f.heads, head = i - t * f.heads, position = q.begin + t;
                for (int pair = lane; pair < half; pair += 64) {
                    Lot v;
                    v.place(pair, f.pairs, f.interleaved);
                    v.set(v.get(f.q + (q.row0 + t) * f.q_token + head * f.q_head));
                    v.turn(Lot::angles(f, position, pair, f.pairs));
                    if (position < 0) v.v[0] = Pair{0.0f, 0.0f};
                    v.store(f.q_out + ((size_t)(q.row0 + t) * f.heads + head) * c.dim);
                }
            }
            continue;
        }
        const int head = task >> 1, side = task & 1, first = max(q.begin, 0), kv_head = head % c.kv_heads;
        if (q.count == 0 || q.length <= first || c.width == 0) continue;
        const uint16_t *const x = (side ? f.v + kv_head * f.v_head : f.k + kv_head * f.k_head) + q.row0 * (side ? f.v_token : f.k_token);
        const int last = min((q.length - 1) / c.page, c.width - 1), fours = c.page / 4, words = c.page * c.dim / 4;
        for (int number = first / c.page + head / c.kv_heads; number <= last; number += slots) {
            const int id = kv_page(c, s, number);
            if (id < 0) continue;
            const int base = number * c.page, lo = max(first, base), hi = min(q.length - base, c.page) + base;
            float *const held = c.scales + ((size_t)id * c.kv_heads + kv_head) * 2 + side;
            uint32_t *const codes = reinterpret_cast<uint32_t *>((side ? c.v : c.k) + ((size_t)id * c.kv_heads + kv_head) * c.page * c.dim);
            const float before = lo > base ? *held : 0.0f;
            uint32_t amax = 0;
            const auto key = [&](Lot &v, const int position, const int pair) {
                v.place(pair, f.pairs, f.interleaved);
                v.set(v.get(x + (position - q.begin) * f.k_token));
                v.turn(Lot::angles(f, position, pair, f.pairs));
            };
            const auto value = [&](const int position, const int d) { return float_of<T>(x[(position - q.begin) * f.v_token + d]); };
            for (int p = lo; p < hi; ++p) {
                if (side) {
                    for (int d = lane; d < c.dim; d += 64) amax = max(amax, magnitude(value(p, d)));
                } else {
                    for (int pair = lane; pair < half; pair += 64) {
                        Lot v;
                        key(v, p, pair);
                        amax = max(amax, v.largest());
                    }
                }
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
            const PageScale to = page_scale(before, amax);
            const bool whole = lo == base || magnitude(to.scale) != magnitude(before);
            const int row_words = c.dim / 4, four0 = (lo - base) / 4, four1 = (hi - base + 3) / 4;
            if (whole) {
                if (lane == 0) *held = to.scale;
                for (int i = lane; i < words; i += 64) {
                    const int t = side ? i % fours : i / row_words;
                    if (side ? t >= four0 && t < four1 : t >= lo - base && t < hi - base) continue;
                    codes[i] = lo > base ? recoded(codes[i], to.ratio) : 0;
                }
            }
            if (side) {
                for (int d = lane; d < c.dim; d += 64) {
                    for (int t4 = four0; t4 < four1; ++t4) {
                        uint32_t *const at = codes + d * fours + t4;
                        uint32_t w = lo == base ? 0 : *at;
                        if (whole) w = recoded(w, to.ratio);
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const int p = base + 4 * t4 + t;
                            if (p >= lo && p < hi) w = (w & ~(0xFFu << (8 * t))) | (uint32_t)(uint8_t)code_of(value(p, d), to.inverse) << (8 * t);
                        }
                        *at = w;
                    }
                }
            } else {
                for (int p = lo; p < hi; ++p) {
                    for (int pair = lane; pair < half; pair += 64) {
                        Lot v;
                        key(v, p, pair);
                        v.store_codes(reinterpret_cast<int8_t *>(codes) + (p - base) * c.dim, to.inverse);
                    }
                }
            }
        }
    }
}

// blockIdx.y: a head; blockIdx.x: a page. The values' codes are turned in the LDS (rows of page + 4 bytes); a thread has eight channels of a token.
template <int T>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvArgs c, const int *page_ids, const int count, uint16_t *k, uint16_t *v)
{
    extern __shared__ int8_t turned[];
    const int head = blockIdx.y, pitch = c.page + 4, eights = c.dim / 8;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const int id = scalars(page_ids)[n];
        const bool in = id >= 0 && id < c.pages;
        const size_t at = ((size_t)(in ? id : 0) * c.kv_heads + head) * c.page * c.dim, to = ((size_t)n * c.kv_heads + head) * c.page * c.dim;
        const float *const held = c.scales + ((size_t)(in ? id : 0) * c.kv_heads + head) * 2;
        const float ks = in ? held[0] : __builtin_nanf(""), vs = in ? held[1] : __builtin_nanf("");
        const auto put = [&](uint16_t *out, const uint32_t a, const uint32_t b, const float scale) {
            v4i w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t from = (e < 2 ? a : b) >> (16 * (e & 1));
                w[e] = (int)round16_pair<T>((float)(int8_t)from * scale, (float)(int8_t)(from >> 8) * scale);
            }
            *reinterpret_cast<v4i *>(out) = in ? w : v4i{(int)(round16<T>(scale) * 0x10001u), (int)(round16<T>(scale) * 0x10001u), (int)(round16<T>(scale) * 0x10001u), (int)(round16<T>(scale) * 0x10001u)};
        };
        __syncthreads();
        for (int i = threadIdx.x * 16; i < c.page * c.dim; i += 256 * 16) {
            const v4i w = *reinterpret_cast<const v4i *>(c.v + at + i);
            int8_t *const row = turned + i / c.page * pitch + i % c.page;
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<int *>(row + 4 * e) = w[e];
        }
        for (int i = threadIdx.x; i < c.page * eights; i += 256) {
            const v2i w = *reinterpret_cast<const v2i *>(c.k + at + (size_t)i * 8);
            put(k + to + (size_t)i * 8, (uint32_t)w[0], (uint32_t)w[1], ks);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < c.page * eights; i += 256) {
            const int t = i / eights, d = (i - t * eights) * 8;
            uint32_t w[2] = {};
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e / 4] |= (uint32_t)(uint8_t)turned[(d + e) * pitch + t] << (8 * (e & 3));
            put(v + to + (size_t)i * 8, w[0], w[1], vs);
        }
    }
}

}  // namespace qm
