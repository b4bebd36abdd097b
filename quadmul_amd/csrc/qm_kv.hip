// C entries of the paged 8-bit cache (include/qm_abi.h): argument checks and launches.
#include <algorithm>
#include <climits>

#include "qm_launch.hpp"
#include "qm_kv.hpp"
#include "qm_attend.hpp"

#define QM_EXPORT extern "C" __attribute__((visibility("default")))

namespace qm {

static bool dim_ok(int dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256; }

// What every call checks of the cache; `tables`: the call looks at the sequences too.
static int check_cache(const qm_kv_cache *c, bool tables)
{
    if (!c) return QM_ERR_NULL;
    if (c->pages < 0 || c->kv_heads < 1 || c->kv_heads > 4096 || !dim_ok(c->head_dim)) return QM_ERR_SHAPE;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return QM_ERR_SHAPE;
    if (c->pages > 0 && (!c->k || !c->v || !c->scales)) return QM_ERR_NULL;
    if ((((uintptr_t)c->k | (uintptr_t)c->v) & 15) || ((uintptr_t)c->scales & 7)) return QM_ERR_ALIGN;
    if (!tables) return QM_OK;
    if (c->sequences < 0 || c->table_width < 0) return QM_ERR_SHAPE;
    if (c->sequences > 0 && (!c->lengths || (c->table_width > 0 && !c->block_table))) return QM_ERR_NULL;
    if (((uintptr_t)c->block_table | (uintptr_t)c->lengths | (uintptr_t)c->query_start) & 3) return QM_ERR_ALIGN;
    return QM_OK;
}
static int check_tokens(const qm_kv_cache *c, int tokens)
{
    if (tokens < 0 || (tokens > 0 && c->sequences == 0)) return QM_ERR_SHAPE;
    return !c->query_start && c->sequences > 0 && tokens % c->sequences != 0 ? QM_ERR_SHAPE : QM_OK;
}
static KvArgs kv_args(const qm_kv_cache *c, int tokens)
{
    return {static_cast<int8_t *>(c->k), static_cast<int8_t *>(c->v), c->scales, c->block_table, c->lengths, c->query_start ? c->query_start : c->lengths, c->pages,
            c->kv_heads, c->page_size, c->head_dim, c->sequences, c->table_width, tokens, c->sequences > 0 ? tokens / c->sequences : 0, c->query_start ? 1 : 0};
}
// The most new tokens of a sequence: what the caller says, inside what is possible. Without a word, packed tokens that are no more than the sequences are
// taken for one each, as a step of a server has them; sequences with more are gone through all the same. 32 sequences of up to 8192 tokens, one new one
// each: attention 38 us, 151 if all of them might be one sequence's; 64 of up to 1000 21 and 34; storing for 64 6.5 and 22. Where they are one
// sequence's: 16 of 4000 115 us and 26, storing 14 and 5.5; 64 442 and 75, 46 and 15.
static int most_new(const qm_kv_cache *c, int tokens, int max_query)
{
    if (c->query_start && max_query <= 0 && tokens <= c->sequences) return 1;
    const int most = c->query_start ? tokens : tokens / std::max(c->sequences, 1);
    return std::max(1, c->query_start && max_query > 0 ? std::min(max_query, most) : most);
}

}  // namespace qm

using namespace qm;

QM_EXPORT int qm_kv_append_i8(const qm_kv_cache *cache, const qm_kv_new *fresh, void *stream)
{
    int st = check_cache(cache, true);
    if (st != QM_OK) return st;
    if (!fresh) return QM_ERR_NULL;
    const qm_kv_new &n = *fresh;
    if (n.dtype != QM_IN_F16 && n.dtype != QM_IN_BF16) return QM_ERR_DTYPE;
    if ((st = check_tokens(cache, n.tokens)) != QM_OK) return st;
    if (n.rotary_pairs < 0 || n.rotary_pairs > cache->head_dim / 2 || n.positions < 0 || (n.rotary_pairs > 0 && n.positions == 0) || (n.q && (n.heads < 1 || (long long)n.tokens * n.heads > INT_MAX))) return QM_ERR_SHAPE;
    if (n.tokens == 0) return QM_OK;
    if (!n.k || !n.v || (n.q && !n.q_out) || (n.rotary_pairs > 0 && (!n.cos || !n.sin))) return QM_ERR_NULL;
    if ((((uintptr_t)n.k | (uintptr_t)n.v | (uintptr_t)n.q | (uintptr_t)n.q_out) & 1) || (((uintptr_t)n.cos | (uintptr_t)n.sin) & 3)) return QM_ERR_ALIGN;
    const KvArgs c = kv_args(cache, n.tokens);
    const KvNewArgs f{static_cast<const uint16_t *>(n.k), static_cast<const uint16_t *>(n.v), static_cast<const uint16_t *>(n.q), static_cast<uint16_t *>(n.q_out),
                      n.k_token_stride, n.k_head_stride, n.v_token_stride, n.v_head_stride, n.q_token_stride, n.q_head_stride, n.cos, n.sin, n.heads,
                      n.rotary_pairs, n.positions, n.interleaved ? 1 : 0};
    const int most = most_new(cache, n.tokens, n.max_query), slots = std::min((most + c.page - 2) / c.page + 1, 4096);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipError_t e;
    // One token of 64 sequences and 8 heads: 17.6 us by workgroups, 7.5 by waves.
    if (most <= 8) {
        const int tasks = slots * 2 * c.kv_heads + (n.q ? std::min(most, 64) * n.heads : 0);
        const auto kernel = n.dtype == QM_IN_F16 ? &kv_append_few_kernel<QM_IN_F16> : &kv_append_few_kernel<QM_IN_BF16>;
        e = enqueue(kernel, dim3((tasks + 3) / 4, std::min(c.sequences, 65535)), dim3(256), 0, s, c, f, slots, tasks);
    } else {
        const bool vector = n.rotary_pairs % 8 == 0;
        const long long items = !n.q ? 0 : vector ? (long long)most * ((n.heads + 1) / 2) * (c.dim / 16) : (long long)most * n.heads * (c.dim / 2);
        const int q_slots = (int)std::min<long long>((items + 2 * c.kv_heads * 256 - 1) / (2 * c.kv_heads * 256), 4096);
        const dim3 grid(slots + q_slots, 2 * c.kv_heads, std::min(c.sequences, 65535));
        const auto kernel = n.dtype == QM_IN_F16 ? (vector ? &kv_append_kernel<QM_IN_F16, true> : &kv_append_kernel<QM_IN_F16, false>)
                                                 : (vector ? &kv_append_kernel<QM_IN_BF16, true> : &kv_append_kernel<QM_IN_BF16, false>);
        e = enqueue(kernel, grid, dim3(256), (size_t)c.page * c.dim, s, c, f, slots);
    }
    return e == hipSuccess ? QM_OK : fail_launch(e);
}

// How a call's work is dealt out: tiles of 16 rows; to a tile and a head a workgroup for each sequence, or all sequences' 64-token
// steps cut into equal parts and joined by a second launch.
namespace {
struct AttendPlan {
    int tiles, rows, wide, parts;
    size_t part_bytes, lse_bytes, bytes;
};
}
static AttendPlan attend_plan(const qm_kv_cache *c, int tokens, int heads, int max_query, int max_length, int window)
{
    AttendPlan p{1, 16, 0, 0, 0, 0, 0};
    if (tokens == 0 || c->sequences == 0) return p;
    const long long most = std::min<long long>((long long)c->table_width * c->page_size, INT_MAX - 2 * ATTEND_STEP);
    long long length = max_length > 0 ? std::min<long long>(max_length, most) : most;
    const int fresh = most_new(c, tokens, max_query);
    if (window > 0) length = std::min<long long>(length, (long long)window + fresh + ATTEND_STEP);
    const int steps = (int)((length + ATTEND_STEP - 1) / ATTEND_STEP);
    const long long rows = (long long)fresh * (heads / c->kv_heads);
    p.tiles = (int)std::min<long long>((rows + 15) / 16, 4096);
    p.rows = (int)std::min<long long>(rows, 16);
    // many rows, and workgroups enough of 64
    if (const long long workgroups = (rows + 63) / 64 * c->kv_heads * c->sequences; rows > 64 && workgroups >= 128) {
        p.wide = workgroups >= 4096 ? 1 : 2;
        p.tiles = (int)std::min<long long>((rows + 63) / 64, 65535);
        return p;
    }
    const long long groups = (long long)p.tiles * c->kv_heads;
    // The second launch costs 5 us, a step of a wave 2 to 3.5, a sequence in one workgroup has its waves go through an eighth of its
    // steps one by one. 32 sequences and 8 heads (256 workgroups): 2048 tokens each 31 us in one piece, 36 cut; 6000 tokens 78 and
    // 82; lengths from 1 to 8192 62 and 41; one sequence of 2048 tokens 15 and 11, of 1024 11 and 11.
    // However many sequences there are, for one of them may be long: one of 131072 tokens and 299 of 200 736 us in one piece, 122 cut; of 16384 150 and
    // 66; 2000 tokens each of 300, 1024 and 2048 sequences 228 and 230, 703 and 706, 1387 and 1387, 5000 of 600 1007 and 1024. (Measured to 4000: one of 16384
    // 944 and 669.)
    if (steps <= 16 || (steps <= 32 && groups * c->sequences >= 128) || c->sequences > 4096) return p;
    // two workgroups of four waves to a CU; a step to a wave at least
    p.parts = (int)std::max<long long>(1, std::min<long long>(512 / groups, (long long)steps * c->sequences / 4));
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    p.part_bytes = (size_t)groups * p.parts * 2 * 16 * c->head_dim * sizeof(float);
    p.lse_bytes = up((size_t)groups * p.parts * 2 * 16 * sizeof(float));
    p.bytes = p.part_bytes + p.lse_bytes + c->sequences * sizeof(int2);
    return p;
}

QM_EXPORT size_t qm_kv_attend_workspace_bytes(const qm_kv_cache *cache, int tokens, int heads, int window, int max_query, int max_length)
{
    if (check_cache(cache, true) != QM_OK || check_tokens(cache, tokens) != QM_OK || heads < 1 || heads % cache->kv_heads != 0) return 0;
    return attend_plan(cache, tokens, heads, max_query, max_length, window).bytes;
}

QM_EXPORT int qm_kv_attend_i8(const qm_kv_cache *cache, const void *q, int dtype, long long q_token_stride, long long q_head_stride, void *out, int tokens,
                              int heads, float scale, int causal, int window, int max_query, int max_length, void *stream, void *workspace,
                              size_t workspace_bytes)
{
    int st = check_cache(cache, true);
    if (st != QM_OK) return st;
    if (dtype != QM_IN_F16 && dtype != QM_IN_BF16) return QM_ERR_DTYPE;
    if ((st = check_tokens(cache, tokens)) != QM_OK) return st;
    if (heads < 1 || heads > 65535 || heads % cache->kv_heads != 0 || window < 0 || (long long)tokens * heads > INT_MAX) return QM_ERR_SHAPE;
    if (tokens == 0) return QM_OK;
    if (!q || !out) return QM_ERR_NULL;
    if ((((uintptr_t)q | (uintptr_t)out) & 1) || ((uintptr_t)workspace & 15)) return QM_ERR_ALIGN;
    const AttendPlan p = attend_plan(cache, tokens, heads, max_query, max_length, window);
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return QM_ERR_SCRATCH;
    uint8_t *const scratch = static_cast<uint8_t *>(workspace);
    const AttendArgs a{static_cast<const uint16_t *>(q), static_cast<uint16_t *>(out), q_token_stride, q_head_stride, heads, causal ? 1 : 0,
                       window > 1 << 30 ? 0 : window, scale * 1.4426950408889634f, p.tiles, p.rows, p.wide, p.parts, reinterpret_cast<float *>(scratch),
                       reinterpret_cast<float *>(scratch + p.part_bytes), reinterpret_cast<int2 *>(scratch + p.part_bytes + p.lse_bytes)};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const KvArgs c = kv_args(cache, tokens);
    const hipError_t e = dtype == QM_IN_F16 ? launch_attend_f16(c, a, s) : launch_attend_bf16(c, a, s);
    return e == hipSuccess ? QM_OK : fail_launch(e);
}

QM_EXPORT int qm_kv_read_i8(const qm_kv_cache *cache, const int *page_ids, int count, int dtype, void *k, void *v, void *stream)
{
    const int st = check_cache(cache, false);
    if (st != QM_OK) return st;
    if (dtype != QM_IN_F16 && dtype != QM_IN_BF16) return QM_ERR_DTYPE;
    if (count < 0) return QM_ERR_SHAPE;
    if (count == 0) return QM_OK;
    if (!page_ids || !k || !v) return QM_ERR_NULL;
    if (((uintptr_t)page_ids & 3) || (((uintptr_t)k | (uintptr_t)v) & 15)) return QM_ERR_ALIGN;
    if (cache->pages == 0) return QM_ERR_SHAPE;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const auto kernel = dtype == QM_IN_F16 ? &kv_read_kernel<QM_IN_F16> : &kv_read_kernel<QM_IN_BF16>;
    const hipError_t e = enqueue(kernel, dim3(std::min(count, 1 << 20), cache->kv_heads), dim3(256), (size_t)cache->head_dim * (cache->page_size + 4), s, kv_args(cache, 0), page_ids, count,
                                 static_cast<uint16_t *>(k), static_cast<uint16_t *>(v));
    return e == hipSuccess ? QM_OK : fail_launch(e);
}
