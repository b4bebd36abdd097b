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
// The four products and two sums are rounded one by one: the codes are defined by them.
__device__ __forceinline__ Pair rotated(const Pair x, const KvNewArgs &f, const int position, const int i, const int pairs)
{
#pragma clang fp contract(off)
    if (i >= pairs) return x;
    const bool in = position < f.positions;
    const size_t at = (size_t)(in ? position : 0) * pairs + i;
    const float c = in ? f.cos[at] : __builtin_nanf(""), s = in ? f.sin[at] : __builtin_nanf("");
    const float ac = x.a * c, bs = x.b * s, bc = x.b * c, as = x.a * s;
    return {ac - bs, bc + as};
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
    return {scale, scale > 0.0f ? 1.0f / scale : 0.0f, scale > 0.0f ? before / scale : 0.0f};
}
__device__ __forceinline__ int code_of(const float scaled) { return (int)fminf(fmaxf(rintf(scaled), -127.0f), 127.0f); }
__device__ __forceinline__ int code_of(const float value, const float factor)
{
#pragma clang fp contract(off)
    return code_of(value * factor);
}

// blockIdx.z: a sequence; blockIdx.y: a head and a side (keys, values) of it; blockIdx.x: below `slots` the pages that the
// sequence's new tokens fall into, past it the rotation of its queries.
template <int T>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvArgs c, const KvNewArgs f, const int slots)
{
    extern __shared__ int8_t image[];  // a page of one head and side
    __shared__ uint32_t largest[4];
    const int tid = threadIdx.x, half = c.dim / 2;
    for (int s = blockIdx.z; s < c.sequences; s += gridDim.z) {
        const KvSequence q = kv_sequence(c, s);
        if ((int)blockIdx.x >= slots) {
            const long long count = (long long)q.count * f.heads * half, stride = (long long)(gridDim.x - slots) * gridDim.y * 256;
            for (long long i = ((long long)(blockIdx.x - slots) * gridDim.y + blockIdx.y) * 256 + tid; i < count; i += stride) {
                const int pair = (int)(i % half), head = (int)(i / half % f.heads), t = (int)(i / half / f.heads);
                const int2 at = pair_at(pair, f.pairs, f.interleaved);
                const uint16_t *const x = f.q + (q.row0 + t) * f.q_token + head * f.q_head;
                Pair v = {float_of<T>(x[at.x]), float_of<T>(x[at.y])};
                v = q.begin + t >= 0 ? rotated(v, f, q.begin + t, pair, f.pairs) : Pair{0.0f, 0.0f};
                uint16_t *const out = f.q_out + ((size_t)(q.row0 + t) * f.heads + head) * c.dim;
                out[at.x] = round16<T>(v.a);
                out[at.y] = round16<T>(v.b);
            }
            continue;
        }
        const int head = blockIdx.y >> 1, side = blockIdx.y & 1, first = max(q.begin, 0);
        if (q.count == 0 || q.length <= first || c.width == 0) continue;
        const int pairs = side ? 0 : f.pairs, steps = side ? c.page : 1;  // a channel's step from token to token, in codes, is 1 or dim
        const uint16_t *const x = side ? f.v + head * f.v_head : f.k + head * f.k_head;
        const long long token = side ? f.v_token : f.k_token;
        const int last = min((q.length - 1) / c.page, c.width - 1);
        for (int number = first / c.page + blockIdx.x; number <= last; number += slots) {
            const int id = kv_page(c, s, number);
            if (id < 0) continue;
            const int base = number * c.page, lo = max(first, base), hi = min(q.length - base, c.page) + base;
            const auto value = [&](const int i) {
                const int pair = i % half, position = lo + i / half;
                const int2 at = pair_at(pair, pairs, f.interleaved);
                const uint16_t *const row = x + (q.row0 + position - q.begin) * token;
                return rotated(Pair{float_of<T>(row[at.x]), float_of<T>(row[at.y])}, f, position, pair, pairs);
            };
            uint32_t amax = 0;
            for (int i = tid; i < (hi - lo) * half; i += 256) {
                const Pair v = value(i);
                amax = max(amax, max(magnitude(v.a), magnitude(v.b)));
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
            __syncthreads();  // (the page before is done with)
            if ((tid & 63) == 0) largest[tid >> 6] = amax;
            __syncthreads();
            amax = max(max(largest[0], largest[1]), max(largest[2], largest[3]));

            float *const held = c.scales + ((size_t)id * c.kv_heads + head) * 2 + side;
            const float before = lo > base ? *held : 0.0f;
            const PageScale to = page_scale(before, amax);
            int8_t *const codes = (side ? c.v : c.k) + ((size_t)id * c.kv_heads + head) * c.page * c.dim;
            const bool whole = lo == base || magnitude(to.scale) != magnitude(before);
            int8_t *const into = whole ? image : codes;
            if (whole) {
                for (int i = tid; i < c.page * c.dim; i += 256) image[i] = lo == base ? 0 : (int8_t)code_of((float)codes[i], to.ratio);
                __syncthreads();  // (and every thread has read the scale)
                if (tid == 0) *held = to.scale;
            }
            for (int i = tid; i < (hi - lo) * half; i += 256) {
                const Pair v = value(i);
                const int2 at = pair_at(i % half, pairs, f.interleaved);
                const int place = lo - base + i / half;
                into[at.x * steps + place * (side ? 1 : c.dim)] = (int8_t)code_of(v.a, to.inverse);
                into[at.y * steps + place * (side ? 1 : c.dim)] = (int8_t)code_of(v.b, to.inverse);
            }
            if (whole) {
                __syncthreads();
                for (int i = tid * 16; i < c.page * c.dim; i += 256 * 16) *reinterpret_cast<v4i *>(codes + i) = *reinterpret_cast<const v4i *>(image + i);
            }
        }
    }
}

// blockIdx.y: a head; blockIdx.x: a page.
template <int T>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvArgs c, const int *page_ids, const int count, uint16_t *k, uint16_t *v)
{
    const int head = blockIdx.y;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        const int id = page_ids[n];
        const bool in = id >= 0 && id < c.pages;
        const size_t at = ((size_t)(in ? id : 0) * c.kv_heads + head) * c.page * c.dim, to = ((size_t)n * c.kv_heads + head) * c.page * c.dim;
        const float *const held = c.scales + ((size_t)(in ? id : 0) * c.kv_heads + head) * 2;
        const float ks = in ? held[0] : __builtin_nanf(""), vs = in ? held[1] : __builtin_nanf("");
        for (int i = threadIdx.x; i < c.page * c.dim; i += 256) {
            k[to + i] = round16<T>(in ? (float)c.k[at + i] * ks : ks);
            v[to + i] = round16<T>(in ? (float)c.v[at + (i % c.dim) * c.page + i / c.dim] * vs : vs);
        }
    }
}

}  // namespace qm
