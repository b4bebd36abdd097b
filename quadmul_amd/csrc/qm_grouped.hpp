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
    int ways = 1;           // up to 16 rows: waves that share a tile of columns
    int chunk = 0;          // K in runs of so many blocks of 32, each summed by workgroups of its own ...
    float *part = nullptr;  // ... which leave their sums here, [runs, M, N], where there are several
};

// Any even K at any address: a wave to a column and four rows, a lane to a byte of B at a time, two elements of each
// row with it. Every scaled element goes into the sum by itself.
constexpr int GROUPED_ROWS = 4;
template <int T, int S>
__global__ __launch_bounds__(256) void gemm_grouped_any_kernel(const GroupedArgs p)
{
    const int lane = threadIdx.x & 63;
    for (long long n = blockIdx.x * 4 + (threadIdx.x >> 6); n < p.N; n += (long long)gridDim.x * 4) {
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
// (v & mask) ^ put in one instruction: a nibble taken out, s turned into s + 8 (its sign bit over) and the exponent put above it
__device__ __forceinline__ uint32_t and_xor(const uint32_t v, const uint32_t mask, const uint32_t put) { return __builtin_amdgcn_bitop3_b32(v, mask, put, 0x6A); }
template <>
struct GroupedWeights<QM_IN_F16> {
    typedef h8 frag;
    static constexpr bool OFFSET = false;
    static __device__ __forceinline__ frag of(const uint32_t w)
    {
        const uint32_t w8 = w >> 8;
        const h2 low = {(_Float16)-1032.0f, (_Float16)-1032.0f}, high = {(_Float16)-72.0f, (_Float16)-72.0f}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
        const auto lower = [](const uint32_t v) { return __builtin_bit_cast(h2, and_xor(v, 0x000F000Fu, 0x64086408u)); };
        const auto upper = [](const uint32_t v) { return __builtin_bit_cast(h2, and_xor(v, 0x00F000F0u, 0x64806480u)); };
        const h2 a = lower(w) + low, b = upper(w) * sixteenth + high, c = lower(w8) + low, d = upper(w8) * sixteenth + high;
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
        const auto pair = [](const uint32_t v) { return (int)and_xor(v, 0x000F000Fu, 0x43084308u); };
        return __builtin_bit_cast(frag, (v4i{pair(w), pair(w >> 4), pair(w >> 8), pair(w >> 12)}));
    }
    static __device__ __forceinline__ frag offset() { return __builtin_bit_cast(frag, (v4i{(int)0xC308C308u, (int)0xC308C308u, (int)0xC308C308u, (int)0xC308C308u})); }  // -136
    static __device__ __forceinline__ v4f mfma(const frag a, const frag b, const v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ int low_halves(const int a, const int b) { return (int)__builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x05040100u); }
__device__ __forceinline__ int high_halves(const int a, const int b) { return (int)__builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x07060302u); }
// eight consecutive elements of x, paired as the nibbles are
__device__ __forceinline__ v4i paired(const v4i x) { return v4i{low_halves(x[0], x[2]), high_halves(x[0], x[2]), low_halves(x[1], x[3]), high_halves(x[1], x[3])}; }

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

// The same from loads in which four lanes side by side have the four blocks of a column, its 64 bytes: the memory pipeline takes 16 bytes of neighbours
// together and of lanes 16 apart each by itself, four times as many accesses. Lane 4 n + j has dwords 0..3 of block
// j of column n; afterwards lane 16 c + 4 b + a has dword c of blocks 0..3 of column 4 a + b.
__device__ __forceinline__ void gather_blocks(uint32_t (&w)[4])
{
    turn_blocks(w);
    const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
    const auto swap = [](uint32_t &a, uint32_t &b, const bool second, const auto neighbour) {
        constexpr int CTRL = decltype(neighbour)::value;
        const uint32_t to_a = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, false), to_b = __builtin_amdgcn_update_dpp(0, (int)a, CTRL, 0xF, 0xF, false);
        a = second ? to_a : a;
        b = second ? b : to_b;
    };
    const std::integral_constant<int, 0xB1> next{};  // lanes 1 0 3 2
    const std::integral_constant<int, 0x4E> over{};  // lanes 2 3 0 1
    swap(w[0], w[1], odd, next);
    swap(w[2], w[3], odd, next);
    swap(w[0], w[2], upper, over);
    swap(w[1], w[3], upper, over);
}
__device__ __forceinline__ int gathered_column(const int r) { return (r & 3) * 4 + (r >> 2); }

// How many scales four blocks have: groups of 128 and its doubles (1), of 64 (2), of 32 (4); any other multiple of 32 (0).
constexpr int group_mode(const int group) { return group % 128 == 0 && (group & (group - 1)) == 0 ? 1 : group == 64 ? 2 : group == 32 ? 4 : 0; }

// Memory that a wave reads through a descriptor: a lane's offset and a shared one to a load, without arithmetic, and zeros past the end.
struct Bytes {
    __amdgpu_buffer_rsrc_t at;
    __device__ __forceinline__ Bytes(const void *p, const size_t size)
        : at(__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)(uint32_t)min(size, (size_t)0xFFFFFFFFu), 0x00020000))
    {
    }
    __device__ __forceinline__ v4i load16(const uint32_t lane, const uint32_t shared) const { return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(at, lane, shared, 0)); }
    __device__ __forceinline__ v2i load8(const uint32_t lane, const uint32_t shared) const { return __builtin_bit_cast(v2i, __builtin_amdgcn_raw_buffer_load_b64(at, lane, shared, 0)); }
    __device__ __forceinline__ uint32_t load4(const uint32_t lane, const uint32_t shared) const { return __builtin_amdgcn_raw_buffer_load_b32(at, lane, shared, 0); }
    __device__ __forceinline__ uint32_t load2(const uint32_t lane, const uint32_t shared) const { return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(at, lane, shared, 0); }
};

// The scales of Q quads of one column, as they are loaded: at(i, run) belongs to block `run` of quad i.
template <int S, int MODE, int Q>
struct GroupedScaleSet {
    static constexpr bool WIDE = S == QM_IN_F32;
    static constexpr int SB = WIDE ? 4 : 2, COUNT = MODE == 0 ? 4 : MODE, ALL = Q * COUNT, WORDS = WIDE || MODE == 0 || ALL == 1 ? ALL : ALL / 2;
    uint32_t raw[WORDS];
    // scale number i of the set, whose first block is number `block` of the row
    static __device__ __forceinline__ int index(const int block, const int i, const int group)
    {
        if constexpr (MODE == 0) return (block + i) * 32 / group;
        else if constexpr (MODE == 1) return (block / 4 + i) >> (__builtin_ctz(group) - 7);
        else return block / (4 / COUNT) + i;
    }
    __device__ __forceinline__ void load(const Bytes &scales, const uint32_t to, const int block, const int group, const int groups)
    {
        // one after the other in memory, and none of them past the end of the row: a load that ends outside the memory gives zeros for all of a word
        const int first = index(block, 0, group);
        if (MODE != 0 && (MODE != 1 || group == 128) && first + ALL <= groups) {
#pragma unroll
            for (int w = 0; w < WORDS; w += 4) {
                const uint32_t at = (uint32_t)(first * SB + w * 4);
                if constexpr (WORDS == 1) {
                    raw[0] = SB * ALL == 4 ? scales.load4(to, at) : scales.load2(to, at);
                } else if constexpr (WORDS == 2) {
                    const v2i v = scales.load8(to, at);
                    raw[0] = (uint32_t)v[0], raw[1] = (uint32_t)v[1];
                } else {
                    const v4i v = scales.load16(to, at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) raw[w + e] = (uint32_t)v[e];
                }
            }
        } else {
            const auto one = [&](const int i) {
                const uint32_t at = (uint32_t)(min(index(block, i, group), groups - 1) * SB);
                return WIDE ? scales.load4(to, at) : scales.load2(to, at);
            };
#pragma unroll
            for (int i = 0; i < WORDS; ++i) raw[i] = WORDS == ALL ? one(i) : one(2 * i) | one(2 * i + 1) << 16;
        }
    }
    // (what turns a loaded scale into a float stays where this is called: moved up to the load, it would wait for it)
    __device__ __forceinline__ void arrive()
    {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) asm("" : "+v"(raw[i]));
    }
    __device__ __forceinline__ float at(const int quad, const int run) const
    {
        const int i = MODE == 1 ? quad : MODE == 2 ? quad * 2 + run / 2 : quad * 4 + run;
        if constexpr (WIDE) return __builtin_bit_cast(float, raw[i]);
        else if constexpr (WORDS == ALL) return float_of<S>((uint16_t)raw[i]);
        else return float_of<S>((uint16_t)(raw[i / 2] >> (16 * (i & 1))));
    }
};

// Up to 16 rows. A workgroup has a run of K (all of it where that fits) of x in its LDS, in the order that the first operand wants it, paired, and goes
// through tiles of columns. A wave has 16 columns and an equal share of the run's quads (four blocks, 64 bytes of each column): `ways` waves share a
// tile, and their sums meet in the LDS. Bound by the weights' way from HBM: two to eight quads of each of 16 waves are in flight, from the next tile too;
// and by what a quad costs of the vector pipeline: about 70 instructions a kilobyte, of which 30 make floats of the weights; 6 TB/s leave it 90.
// (With x from the L2 by each wave for itself, 4 KiB of x for a KiB or two of weights, 13 x 8192 x 28672 took 52 us; with x put into the LDS
// by 832 workgroups 45; now 37 with the sum of its seven runs, 3.3 TB/s. 1 x 4096 x 4096 5.1, 1 x 28672 x 4096 in groups of 32 20.)
template <int T, int S, int MODE, int NW>
__global__ __launch_bounds__(NW * 64, 4) void gemm_grouped_rows_kernel(const GroupedArgs p)
{
    typedef GroupedWeights<T> W;
    typedef typename W::frag frag;
    // SET: quads that are loaded at a time, one set ahead; PER: blocks of one scale
    constexpr int SET = MODE == 1 || MODE == 2 ? 4 : 2, RING = 2, PER = MODE == 1 ? 4 : MODE == 2 ? 2 : 1;
    typedef GroupedScaleSet<S, MODE, SET> Scales;
    extern __shared__ v4i staged[];
    __shared__ v4f sums[NW][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, c = lane >> 4;
    const int block0 = blockIdx.y * p.chunk, blocks = min(p.chunk, p.K / 32 - block0), quads = (blocks + 3) / 4;
    const int pitch = p.M | 1;                                                           // rows of 16 bytes for eight k
    v4f *const offsets = reinterpret_cast<v4f *>(staged + (size_t)p.chunk * 4 * pitch);  // -136 times the sums of x, for each scale and four rows

    // the waves' tiles, side by side; a wave's turns: sets of four quads of one tile after the other
    const int abreast = NW / p.ways, groups = ((p.N + 15) / 16 + abreast - 1) / abreast;
    const int each = (quads + p.ways - 1) / p.ways, quad0 = min(wave % p.ways * each, quads), quad1 = min(quad0 + each, quads);
    const int sets = (quad1 - quad0 + SET - 1) / SET, mine = ((int)blockIdx.x < groups ? (groups - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0);
    const auto column0 = [&](const int group) { return (group * abreast + wave / p.ways) * 16; };
    // (columns past the last one, and blocks past the end of K in the last row, are zeros past the end)
    const uint32_t w_at = (lane >> 2) * (uint32_t)(p.K / 2) + 16 * (lane & 3), s_at = gathered_column(r) * (uint32_t)(p.groups * Scales::SB);
    const size_t w_all = (size_t)p.N * (p.K / 2), s_all = (size_t)p.N * p.groups * Scales::SB;
    struct Set {
        v4i w[SET];
        Scales s;
    };
    int load_group = blockIdx.x, load_quad = quad0;
    const auto load = [&](Set &to) {
        const int n0 = column0(load_group);
        const size_t w_from = min((size_t)n0 * (p.K / 2) + (size_t)block0 * 16, w_all), s_from = min((size_t)n0 * p.groups * Scales::SB, s_all);
        const Bytes weights(p.B + w_from, w_all - w_from), scales(static_cast<const uint8_t *>(p.scale) + s_from, s_all - s_from);
#pragma unroll
        for (int i = 0; i < SET; ++i) to.w[i] = weights.load16(w_at, (load_quad + i) * 64);
        to.s.load(scales, s_at, block0 + load_quad * 4, p.group, p.groups);
        load_quad += SET;
        if (load_quad >= quad1) load_quad = quad0, load_group += gridDim.x;
    };

    // x first, for it is waited for first (four loads of a thread at a time); the weights are in flight while it is put in place
    constexpr int BATCH = 4, THREADS = NW * 64;
    const int units = quads * 16, all = units * p.M;
    v4i x[BATCH];
    const auto get = [&](const int from) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int at = min(from + i * THREADS + (int)threadIdx.x, all - 1), m = at / units, k = min(at - m * units, blocks * 4 - 1);
            if (from + i * THREADS < all) x[i] = *reinterpret_cast<const v4i_half_aligned *>(p.x + m * p.x_stride + (size_t)(block0 * 4 + k) * 8);
        }
    };
    const auto put_in_place = [&](const int from) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int at = from + i * THREADS + (int)threadIdx.x, m = at / units, k = at - m * units;
            if (at < all) staged[k * pitch + m] = k < blocks * 4 ? paired(x[i]) : v4i{};
        }
    };
    get(0);
    Set ring[RING];
    const int turns = mine * sets;
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
        if (i < turns) load(ring[i]);
    put_in_place(0);
    for (int from = BATCH * THREADS; from < all; from += BATCH * THREADS) {
        get(from);
        put_in_place(from);
    }
    __syncthreads();
    const v4i *const my_x = staged + c * pitch + min(r, p.M - 1);
    const auto x_frag = [&](const int block) { return __builtin_bit_cast(frag, my_x[block * 4 * pitch]); };
    if constexpr (W::OFFSET) {
        for (int i = wave; i < quads * 4 / PER; i += NW) {
            v4f sum = {};
#pragma unroll
            for (int j = 0; j < PER; ++j) sum = W::mfma(x_frag(i * PER + j), W::offset(), sum);
            if (r == 0) offsets[i * 4 + c] = sum;
        }
        __syncthreads();
    }

    v4f total = {};
    const auto use = [&](Set &in, const int quad) {
        in.s.arrive();
#pragma unroll
        for (int q = 0; q < SET; ++q) {
            if (quad + q >= quad1) break;
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (uint32_t)in.w[q][i];
            gather_blocks(w);
#pragma unroll
            for (int run = 0; run < 4; run += PER) {
                v4f part = {};
                if constexpr (W::OFFSET) part = offsets[((quad + q) * 4 + run) / PER * 4 + c];
#pragma unroll
                for (int i = run; i < run + PER; ++i) part = W::mfma(x_frag((quad + q) * 4 + i), W::of(w[i]), part);
                total += part * in.s.at(q, run);
            }
        }
    };
    const auto put = [&](const int m, const int column, const float v) {
        if (m >= p.M || column >= p.N) return;
        if (p.part != nullptr) p.part[((size_t)blockIdx.y * p.M + m) * p.N + column] = v;
        else p.D[(size_t)m * p.N + column] = round16<T>(p.bias != nullptr ? v + float_of<T>(p.bias[column]) : v);
    };
    const auto finish = [&](const int group) {
        if (p.ways == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) put(4 * c + i, column0(group) + gathered_column(r), total[i]);
        } else {
            __syncthreads();  // (the group before is read)
            sums[wave][lane] = total;
            __syncthreads();
            for (int i = threadIdx.x; i < abreast * 256; i += THREADS) {
                const int tile = i >> 8, column = i & 15, m = (i >> 4) & 15;
                float v = 0.0f;
                for (int w = 0; w < p.ways; ++w) v += sums[tile * p.ways + w][gathered_column(column) + 16 * (m >> 2)][m & 3];  // (its own inverse)
                put(m, (group * abreast + tile) * 16 + column, v);
            }
        }
        total = v4f{};
    };
    int group = blockIdx.x, quad = quad0;
    for (int done = 0; done < turns; done += RING) {
#pragma unroll
        for (int i = 0; i < RING; ++i) {
            if (done + i >= turns) break;
            if (done + i + RING - 1 < turns) load(ring[(i + RING - 1) % RING]);
            use(ring[i], quad);
            quad += SET;
            if (quad >= quad1) {
                finish(group);
                quad = quad0, group += gridDim.x;
            }
        }
    }
    if (sets == 0)  // (a share of nothing: the others wait for it)
        for (; group < groups; group += gridDim.x) finish(group);
}

// The sums of the runs of K into one, always in the same order.
template <int T>
__global__ __launch_bounds__(256) void gemm_grouped_join_kernel(const GroupedArgs p, const int runs)
{
    const size_t all = (size_t)p.M * p.N;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        float v = 0.0f;
#pragma unroll 8
        for (int run = 0; run < runs; ++run) v += p.part[run * all + i];
        p.D[i] = round16<T>(p.bias != nullptr ? v + float_of<T>(p.bias[i % p.N]) : v);
    }
}

// 17 to 64 rows: tiles of 16 MT rows and 64 NT columns, a step of four blocks (128 elements of K) at a time. x goes through the LDS, two steps of it, in
// the order of the first operand; a wave makes the second operand of its 16 NT columns itself, from 64 bytes of each, for all rows. The sums
// over a group and those over all of K are in registers of their own. Bound by the instructions that make floats of the weights (46
// for 16 columns and a step) until there are 64 rows, whose matrix instructions take as long.
// A row's 16 pieces of a step are dealt to the places r ^ piece, so that neither writing 16 of one row nor reading one of 16 rows meets a bank twice.
template <int T, int S, int MODE, int MT, int NT>
__global__ __launch_bounds__(256, 2) void gemm_grouped_tile_kernel(const GroupedArgs p)
{
    typedef GroupedWeights<T> W;
    typedef typename W::frag frag;
    typedef GroupedScaleSet<S, MODE, 1> Scales;
    constexpr int PER = MODE == 1 ? 4 : MODE == 2 ? 2 : 1, BM = 16 * MT, BN = 64 * NT, PIECES = BM / 16;  // PIECES: of x, 16 bytes each, of a thread and step
    __shared__ v4i staged[2][4 * BM * 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, c = lane >> 4;
    const int block0 = blockIdx.z * p.chunk, blocks = min(p.chunk, p.K / 32 - block0), quads = (blocks + 3) / 4;
    const int m0 = blockIdx.x * BM, n0 = blockIdx.y * BN + wave * 16 * NT;

    const size_t w_all = (size_t)p.N * (p.K / 2), s_all = (size_t)p.N * p.groups * Scales::SB;
    const size_t w_from = min((size_t)n0 * (p.K / 2) + (size_t)block0 * 16, w_all), s_from = min((size_t)n0 * p.groups * Scales::SB, s_all);
    const Bytes weights(p.B + w_from, w_all - w_from), scales(static_cast<const uint8_t *>(p.scale) + s_from, s_all - s_from);
    const uint32_t w_at = (lane >> 2) * (uint32_t)(p.K / 2) + 16 * (lane & 3), s_at = gathered_column(r) * (uint32_t)(p.groups * Scales::SB);
    struct Step {
        v4i w[NT];
        Scales s[NT];
    };
    const auto load = [&](Step &to, const int quad) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            to.w[t] = weights.load16(w_at + t * 16 * (uint32_t)(p.K / 2), quad * 64);
            to.s[t].load(scales, s_at + t * 16 * (uint32_t)(p.groups * Scales::SB), block0 + quad * 4, p.group, p.groups);
        }
    };
    // piece `threadIdx.x % 16` of rows threadIdx.x / 16 and every sixteenth from there on
    const int piece = threadIdx.x & 15, my_row = threadIdx.x >> 4;
    v4i x[PIECES];
    const auto get = [&](const int quad) {
        const uint16_t *const at = p.x + (size_t)(block0 * 4 + min(quad * 16 + piece, blocks * 4 - 1)) * 8;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) x[i] = *reinterpret_cast<const v4i_half_aligned *>(at + min(m0 + my_row + 16 * i, p.M - 1) * p.x_stride);
    };
    const auto put_in_place = [&](const int quad) {
        const bool in = quad * 16 + piece < blocks * 4;  // past the end of K: zeros, which whatever follows the weights meets
        v4i *const to = staged[quad & 1] + (piece >> 2) * (BM * 4) + (piece & 3) * 16 + (my_row ^ piece);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) to[i * 64] = in ? paired(x[i]) : v4i{};
    };

    v4f total[MT][NT] = {};
    const auto use = [&](Step &in, const int quad) {
        uint32_t w[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            in.s[t].arrive();
#pragma unroll
            for (int i = 0; i < 4; ++i) w[t][i] = (uint32_t)in.w[t][i];
            gather_blocks(w[t]);
        }
        const v4i *const from = staged[quad & 1] + c * 16;
#pragma unroll
        for (int run = 0; run < 4; run += PER) {
            v4f part[MT][NT];
#pragma unroll
            for (int i = run; i < run + PER; ++i) {
                frag xs[MT], ws[NT];
#pragma unroll
                for (int a = 0; a < MT; ++a) xs[a] = __builtin_bit_cast(frag, from[i * (BM * 4) + a * 64 + (r ^ (4 * i + c))]);
#pragma unroll
                for (int t = 0; t < NT; ++t) ws[t] = W::of(w[t][i]);
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    if (i == run) {
                        v4f first = {};
                        if constexpr (W::OFFSET) first = W::mfma(xs[a], W::offset(), first);
#pragma unroll
                        for (int t = 0; t < NT; ++t) part[a][t] = W::mfma(xs[a], ws[t], first);
                    } else {
                        // (a run's later offsets: into the first column's sum they cannot go, the others need them too)
                        v4f first = {};
                        if constexpr (W::OFFSET) first = W::mfma(xs[a], W::offset(), first);
#pragma unroll
                        for (int t = 0; t < NT; ++t) part[a][t] = W::mfma(xs[a], ws[t], W::OFFSET ? part[a][t] + first : part[a][t]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float scale = in.s[t].at(0, run);
#pragma unroll
                for (int a = 0; a < MT; ++a) total[a][t] += part[a][t] * scale;
            }
        }
    };

    Step one, two;
    get(0);
    load(one, 0);
    put_in_place(0);
    get(min(1, quads - 1));
    for (int quad = 0; quad < quads; quad += 2) {
        __syncthreads();
        put_in_place(quad + 1);  // (past the last step: zeros that nobody reads)
        get(min(quad + 2, quads - 1));
        load(two, min(quad + 1, quads - 1));
        use(one, quad);
        if (quad + 1 >= quads) break;
        __syncthreads();
        put_in_place(quad + 2);
        get(min(quad + 3, quads - 1));
        load(one, min(quad + 2, quads - 1));
        use(two, quad + 1);
    }

#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = n0 + 16 * t + gathered_column(r);
        const float bias = p.bias != nullptr && p.part == nullptr && n < p.N ? float_of<T>(p.bias[n]) : 0.0f;
#pragma unroll
        for (int a = 0; a < MT; ++a) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = m0 + a * 16 + 4 * c + i;
                if (m < p.M && n < p.N) {
                    if (p.part != nullptr) p.part[((size_t)blockIdx.z * p.M + m) * p.N + n] = total[a][t][i];
                    else p.D[(size_t)m * p.N + n] = round16<T>(p.bias != nullptr ? total[a][t][i] + bias : total[a][t][i]);
                }
            }
        }
    }
}

// Eight weights as 16-bit floats in the order they have in memory, exactly.
template <int T>
__device__ __forceinline__ v4i plain_weights(const uint32_t w)
{
    if constexpr (T == QM_IN_F16) {
        const v4i v = __builtin_bit_cast(v4i, GroupedWeights<T>::of(w));
        return v4i{low_halves(v[0], v[1]), low_halves(v[2], v[3]), high_halves(v[0], v[1]), high_halves(v[2], v[3])};
    }
    v4i out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto value = [&](const int k) { return __builtin_bit_cast(int, (float)((int)(w << (28 - 4 * k)) >> 28)); };
        out[i] = high_halves(value(2 * i), value(2 * i + 1));  // (the float of a small integer has zeros below)
    }
    return out;
}

// Many rows: tiles of 16 WM MT rows and 16 WN NT columns, a step of two blocks (64 elements of K) at a time. x and the weights, as floats, go
// through the LDS, two steps of them, each weight made a float once by one thread of the workgroup; a wave has 16 MT rows and 16 NT columns.
// Bound by what the matrix cores (16 cycles an instruction, 41 % of the time) and the vector pipeline (33 %: the sums times their scales, and
// making floats) do not do at the same time. 2048 x 11008 x 4096 in groups of 128: 214 us, 863 TFLOP/s; with each wave making floats of
// its own columns 274, without one half of the waves preparing before and the other after 226, as four waves to each of two workgroups of a CU
// 241. Groups of 64 305 us, of 32 335.
// Piece p (eight k) of row r lies at p * rows + (r ^ p): neither eight pieces of a row, written together, nor a piece of eight rows, read
// together, meet a bank twice.
template <int T, int S, int MODE, int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_grouped_wide_kernel(const GroupedArgs p)
{
    typedef GroupedWeights<T> W;
    typedef typename W::frag frag;
    constexpr int THREADS = 64 * WM * WN, BM = 16 * WM * MT, BN = 16 * WN * NT, XP = BM * 8 / THREADS, WP = (BN * 4 + THREADS - 1) / THREADS;
    constexpr int SCALES = MODE == 1 || MODE == 2 ? 1 : 2;  // of a step; or one
    constexpr bool TWO = MODE == 1;                         // for two steps
    extern __shared__ v4i staged[];
    v4i *const all_x = staged, *const all_w = staged + 2 * 8 * BM;
    float *const all_s = reinterpret_cast<float *>(staged + 2 * 8 * (BM + BN));
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, c = lane >> 4;
    const int block0 = blockIdx.z * p.chunk, blocks = min(p.chunk, p.K / 32 - block0), steps = (blocks + 1) / 2;
    const int m0 = blockIdx.x * BM, n0 = blockIdx.y * BN;

    const uint16_t *x_at[XP];
    const uint8_t *w_at[WP];
#pragma unroll
    for (int i = 0; i < XP; ++i) x_at[i] = p.x + min(m0 + tid / 8 + i * (THREADS / 8), p.M - 1) * p.x_stride + (size_t)block0 * 32;
#pragma unroll
    for (int i = 0; i < WP; ++i) w_at[i] = p.B + (size_t)min(n0 + tid / 4 + i * (THREADS / 4), p.N - 1) * (p.K / 2) + (size_t)block0 * 16;
    const int s_block = SCALES == 2 ? tid / BN : 0;
    const size_t s_row = (size_t)min(n0 + tid % BN, p.N - 1) * p.groups;

    struct Raw {
        v4i x[XP];
        v2i w[WP];
        uint32_t s;
    };
    const auto get = [&](Raw &to, int step) {
        step = min(step, steps - 1);
        const int k = min(step * 64 + (tid & 7) * 8, blocks * 32 - 8), half = min(step * 4 + (tid & 3), blocks * 2 - 1);
#pragma unroll
        for (int i = 0; i < XP; ++i) to.x[i] = *reinterpret_cast<const v4i_half_aligned *>(x_at[i] + k);
#pragma unroll
        for (int i = 0; i < WP; ++i) to.w[i] = *reinterpret_cast<const v2i *>(w_at[i] + half * 8);
        if (tid < BN * SCALES) {
            const size_t at = s_row + min((block0 + step * 2 + s_block) * 32 / p.group, p.groups - 1);
            to.s = S == QM_IN_F32 ? static_cast<const uint32_t *>(p.scale)[at] : static_cast<const uint16_t *>(p.scale)[at];
        }
    };
    const auto put_in_place = [&](const Raw &from, const int step) {
        v4i *const to_x = all_x + (step & 1) * (8 * BM), *const to_w = all_w + (step & 1) * (8 * BN);
        const int piece = tid & 7, row = tid / 8, half = tid & 3, column = tid / 4;
        const bool in = step * 8 + piece < blocks * 4;  // past the end of K: zeros, which whatever weights meet
#pragma unroll
        for (int i = 0; i < XP; ++i) to_x[piece * BM + i * (THREADS / 8) + (row ^ piece)] = in ? from.x[i] : v4i{};
#pragma unroll
        for (int i = 0; i < WP; ++i) {
            if (BN * 4 < THREADS && tid >= BN * 4) break;
#pragma unroll
            for (int j = 0; j < 2; ++j) to_w[(2 * half + j) * BN + i * (THREADS / 4) + (column ^ (2 * half + j))] = plain_weights<T>((uint32_t)from.w[i][j]);
        }
        if (tid < BN * SCALES) all_s[(step & 1) * (BN * SCALES) + tid] = S == QM_IN_F32 ? __builtin_bit_cast(float, from.s) : float_of<S == QM_IN_F32 ? QM_IN_F16 : S>((uint16_t)from.s);
    };

    v4f total[MT][NT] = {}, part[MT][NT];
    const int wm = wave % WM, wn = wave / WM;
    const auto use = [&](const int step, const bool first, const bool last) {
        const v4i *const from_x = all_x + (step & 1) * (8 * BM) + wm * (16 * MT), *const from_w = all_w + (step & 1) * (8 * BN) + wn * (16 * NT);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            frag xs[MT], ws[NT];
            const int piece = 4 * b + c;
#pragma unroll
            for (int a = 0; a < MT; ++a) xs[a] = __builtin_bit_cast(frag, from_x[piece * BM + 16 * a + (r ^ piece)]);
#pragma unroll
            for (int t = 0; t < NT; ++t) ws[t] = __builtin_bit_cast(frag, from_w[piece * BN + 16 * t + (r ^ piece)]);
            const bool fresh = SCALES == 2 || (b == 0 && first), full = SCALES == 2 || (b == 1 && last);
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int t = 0; t < NT; ++t) part[a][t] = W::mfma(xs[a], ws[t], fresh ? v4f{} : part[a][t]);
            if (full) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float scale = all_s[(step & 1) * (BN * SCALES) + (SCALES == 2 ? b * BN : 0) + wn * (16 * NT) + 16 * t + r];
#pragma unroll
                    for (int a = 0; a < MT; ++a) total[a][t] += part[a][t] * scale;
                }
                __builtin_amdgcn_sched_barrier(0);  // (two sets of sums at a time would not fit)
            }
        }
    };

    // One half of the waves, one of the two of each SIMD, prepares the next step before it multiplies, the other after: the vector pipeline and the
    // matrix cores have something to do at the same time.
    const bool early = wave < WM * WN / 2;
    Raw raw[2];
    get(raw[0], 0);
    put_in_place(raw[0], 0);
    get(raw[1], 1);
    for (int step = 0; step < steps; step += 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            __syncthreads();
            const auto prepare = [&] {
                if (step + i < steps) put_in_place(raw[i ^ 1], step + i + 1);
                get(raw[i], step + i + 2);
            };
            if (early) prepare();
            use(step + i, !TWO || i == 0, !TWO || i == 1);  // (the second may be past the end of K: zeros)
            __builtin_amdgcn_sched_barrier(0);
            if (!early) prepare();
        }
    }

#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = n0 + (wn * NT + t) * 16 + r;
        const float bias = p.bias != nullptr && p.part == nullptr && n < p.N ? float_of<T>(p.bias[n]) : 0.0f;
#pragma unroll
        for (int a = 0; a < MT; ++a) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = m0 + (wm * MT + a) * 16 + 4 * c + i;
                if (m < p.M && n < p.N) {
                    if (p.part != nullptr) p.part[((size_t)blockIdx.z * p.M + m) * p.N + n] = total[a][t][i];
                    else p.D[(size_t)m * p.N + n] = round16<T>(p.bias != nullptr ? total[a][t][i] + bias : total[a][t][i]);
                }
            }
        }
    }
}

}  // namespace qm
