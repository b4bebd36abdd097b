// C entries of the mixture of experts (include/qm_abi.h): argument checks, choice of kernels, launches.
#include <algorithm>
#include <climits>

#include "../../include/qm_abi.h"
#include "qm_launch.hpp"
#include "qm_experts.hpp"
#include "qm_experts_sort.hpp"
#include "qm_route.hpp"

#define QM_EXPORT extern "C" __attribute__((visibility("default")))

namespace qm {

static int check_sizes(const qm_expert_weights *w, const int dtype)
{
    if (!w) return QM_ERR_NULL;
    if (w->scale_dtype != QM_IN_F32 && w->scale_dtype != dtype) return QM_ERR_DTYPE;
    return w->experts < 0 || w->n < 0 || w->k < 0 || (w->k & 1) || w->group < 32 || w->group % 32 != 0 ? QM_ERR_SHAPE : QM_OK;
}
static int check_weights(const qm_expert_weights *w, const int dtype)
{
    if (const int e = check_sizes(w, dtype); e != QM_OK) return e;
    if (w->experts > 0 && w->n > 0 && w->k > 0 && (!w->weight || !w->scale)) return QM_ERR_NULL;
    return ((uintptr_t)w->scale & (w->scale_dtype == QM_IN_F32 ? 3 : 1)) || ((uintptr_t)w->bias & 1) ? QM_ERR_ALIGN : QM_OK;
}

static size_t up256(const size_t n) { return (n + 255) / 256 * 256; }

// `across`: tiles that the columns of the (an MLP's first) product with experts_tile_kernel are; k, group: that product's.
static ExpertsPlan experts_plan(const bool mlp, const int tokens, const int top_k, const int experts, const int across, const int k, const int group, size_t at)
{
    const int slots = tokens * top_k;
    ExpertsPlan p{};
    p.bytes = at;
    if (slots == 0 || experts == 0 || experts > EXPERTS_SORTED) return p;
    const auto mean = [&](const int rows) { return slots >= (long long)rows * experts; };
    // Up to 16 rows, by the mean number of an expert's rows (some have several times the mean), are for experts_rows_kernel; tiles of 32 and 64 want work for the chip too. us of the MLP:
    // rows of a tile in front (a slash: parts of K in the second product), "wide" 8 experts, 2 of them, 4096 x 14336, float16, groups of 128; "odd" the same of 4096 x 11008, bf16, groups of 32;
    // "narrow" 128, 8, 2048 x 1024, bf16, 128; "64" 6 of 64, 2048 x 1408, float16, 32; "short" 4 of 16, 4096 x 1024, bf16, 64.
    //   mean 4    wide   8: 159, 16: 175, 32/2: 220;   narrow  8: 98, 16: 114, 32: 110
    //   mean 6    narrow  16: 131, 32: 117              mean 8    wide  16: 203, 32/2: 223;   narrow  16: 132, 32: 115;   64 (mean 9)  16: 134, 32: 143
    //   mean 12   wide  16: 241, 32/2: 226, 64/2: 239;   odd  16: 228, 32/2: 286;   64  16: 148, 32: 144
    //   mean 16   wide  16: 283, 32/2: 259, 64/2: 241;   odd  16: 302, 32/8: 344, 64/2: 302;   narrow  16: 183, 32: 133, 64: 148;   short  16: 52, 32: 73, 64: 89
    //   mean 32   wide  32/4: 281, 64/2: 249;   odd  16: 475, 32/4: 379, 64/2: 313;   narrow  32: 164, 64: 176;   short  16: 79, 32: 80, 64: 93
    //   mean 48   64  32: 239, 64: 206;   narrow  32: 198, 64: 209;   short  32: 82, 64: 100      mean 64   wide  32/4: 407, 64/4: 353;   short  32: 104, 64: 103
    const long long work = (long long)slots * across, filled = (long long)std::min(experts, slots) * across;
    // One product, "down" 8 experts, 2 of them, 4096 x 11008 (K), bf16, "up" 11008 x 4096, "short" 4 of 16, 4096 x 1024, "64" 6 of 64, 2048 x 1408, groups of 32:
    //   mean 8    down  16: 54, 32/2: 88;   up  16: 55, 32: 70;   short  16: 19, 32: 21        mean 12   64  16: 55, 32: 42, 64: 52
    //   mean 16   down  16: 80, 32/2: 114, 64/2: 98;   up  16: 79, 32: 73, 64/2: 78            mean 32   down  16: 132, 32/2: 116, 64/2: 99;   short  16: 34, 32: 27, 64: 31
    //   mean 64   down  32/4: 146, 64/4: 131;   up  32: 117, 64/2: 117;   short  32: 31, 64: 37      mean 128   up  32: 169, 64/2: 163;   short  32: 47, 64: 61
    //   mean 512  up  32: 517, 64: 458;   short  32: 127, 64: 138
    const bool tiles = mean(32) || (mean(6) && (mlp ? filled >= 1024 || work >= (group % 64 == 0 ? 8192 : 10240) : work >= 4096));
    const bool high = mlp ? mean(64) || (filled >= 512 && mean(k >= 4096 ? 16 : 48)) : mean(k >= 8192 ? 16 : k >= 4096 ? 64 : 1024);
    p.rows = tiles ? high ? 64 : 32 : mean(6) ? 16 : mean(3) ? 8 : tokens > 2 ? 4 : 2;
    p.tiles = slots / p.rows + std::min(experts + 1, slots);
    p.order = at;
    p.list = p.order + up256((size_t)slots * 4);
    p.count = p.list + up256((size_t)p.tiles * 16);
    p.bytes = p.count + 256;
    return p;
}
// The slots sorted (where `slots` is not 0) and x made ready (where it has rows).
static hipError_t sort_slots(const ExpertsPlan &plan, const int *chosen, const int slots, const int experts, const ExpertsReady &ready, const int dtype, char *at, hipStream_t s)
{
    const int grid = (slots > 0 ? 1 : 0) + (int)std::min((ready.rows + 15ll) / 16, 4096ll);
    return enqueue(dtype == QM_IN_F16 ? &experts_sort_kernel<QM_IN_F16> : &experts_sort_kernel<QM_IN_BF16>, dim3(grid), dim3(1024), (size_t)(experts + 1) * 4, s, chosen, slots, experts, plan.rows,
                   reinterpret_cast<int *>(at + plan.order), reinterpret_cast<int *>(at + plan.list), reinterpret_cast<int *>(at + plan.count), ready);
}

static ExpertsArgs args_of(const qm_expert_weights *w, const void *x, const long long x_token, const long long x_choice, const int *chosen, void *out, const int tokens, const int top_k,
                           const ExpertsPlan &plan, const char *at)
{
    ExpertsArgs p{};
    // (the distance of rows of which there is only one says nothing)
    p.x = static_cast<const uint16_t *>(x), p.x_token = tokens > 1 ? x_token : 0, p.x_choice = top_k > 1 ? x_choice : 0, p.chosen = chosen;
    p.B = static_cast<const uint8_t *>(w->weight), p.scale = w->scale, p.bias = static_cast<const uint16_t *>(w->bias), p.out = out;
    p.slots = tokens * top_k, p.top_k = top_k, p.experts = w->experts, p.N = w->n, p.K = w->k, p.group = w->group;
    p.groups = (int)(((long long)w->k + w->group - 1) / w->group);
    p.magic = w->group == 32 ? 0u : (uint32_t)(((1ull << 32) + w->group / 32 - 1) / (w->group / 32));
    p.top_k_magic = ((1ull << 32) + top_k - 1) / top_k;
    p.order = reinterpret_cast<const int *>(at + plan.order), p.tiles = reinterpret_cast<const int *>(at + plan.list), p.count = reinterpret_cast<const int *>(at + plan.count);
    return p;
}

static bool tiles_take(const int k) { return k > 0 && k % 32 == 0 && k < 1 << 20; }
// Which kernel runs a product. The matrix cores want a K of whole blocks, weights at sixteen bytes, offsets of 32 bits from an expert's first weight and scale, and block
// numbers below 2^15 for the division by the size of a group; the kernel for few rows, rows of x at sixteen bytes too and offsets of 32 bits from the first one.
static ExpertsKernel kernel_of(const ExpertsArgs &p, const ExpertsPlan &plan)
{
    if (!tiles_take(p.K) || ((uintptr_t)p.B & 15) != 0 || plan.rows == 0 || p.N > 65535 * 32) return EXPERTS_ANY;
    if ((unsigned long long)p.N * std::max(p.K / 2, p.groups * 4) >= 1ull << 32) return EXPERTS_ANY;
    const long long last = (p.slots / p.top_k - 1) * p.x_token + (p.top_k - 1) * p.x_choice + p.K;
    const bool rows = ((uintptr_t)p.x & 15) == 0 && p.x_token % 8 == 0 && p.x_choice % 8 == 0 && last < 1ll << 31;
    if (plan.rows <= 16 && rows && (long long)p.slots * p.top_k < 1ll << 32 && (long long)plan.tiles * ((p.N + 15) / 16) < 1ll << 31) return EXPERTS_ROWS;
    // (a launch has less than 2^32 threads: more than 100 GB of products)
    return (long long)plan.tiles * ((p.N + 127) / 128) < 1ll << 24 ? EXPERTS_TILES : EXPERTS_ANY;
}
// Room for x made ready: its rows and a float for each; none where K is not for the tiles.
static size_t ready_bytes(const size_t rows, const int k) { return tiles_take(k) ? up256(rows * ready_stride(k) * 2) + up256(rows * 4) : 0; }
static ExpertsReady make_ready(ExpertsArgs &p, const int dtype, void *to)
{
    p.shared = p.x_choice == 0;
    const int rows = p.shared ? p.slots / p.top_k : p.slots;
    float *const back = reinterpret_cast<float *>(static_cast<char *>(to) + up256((size_t)rows * ready_stride(p.K) * 2));
    p.ready = static_cast<const uint16_t *>(to), p.back = dtype == QM_IN_BF16 ? back : nullptr;
    return {p.x, p.x_token, p.x_choice, p.shared ? 1 : p.top_k, rows, p.K, static_cast<uint16_t *>(to), back};
}
// Up to 64 slots the kernel for few rows finds its tiles by itself: 8 tokens, 8 of 128 of 2048 x 1024, 34.8 us, 36.8 with the slots sorted first; 1 token 13.3, 15.9.
static bool sorts(const ExpertsKernel kernel, const int slots) {
    return kernel == EXPERTS_TILES || (kernel == EXPERTS_ROWS && slots > 64); }
static hipError_t launch_product(ExpertsArgs p, const ExpertsKernel kernel, const ExpertsPlan &plan, const int dtype, const int scale_dtype, const ExpertsOut out, hipStream_t s)
{
    if (!sorts(kernel, p.slots)) p.order = nullptr;
    return (dtype == QM_IN_F16 ? launch_experts_f16 : launch_experts_bf16)(p, plan, scale_dtype, out, kernel, s);
}

// Into how many parts K is cut for a product (of an MLP the second) whose tiles are not enough for the chip, at least 1024 of K to each: for a workgroup to a CU, or two where tiles of 64 rows are filled. us of
// "wide" as above with 1, 2, 4, 8 parts: mean 16 295, 241, 252, 260; 32 303, 249, 266, 273; 48 327, 317, 292, 290; 64 385, 374, 353, 372; 128 585, 537, 548, 590.
static int splits_of(const int rows, const int slots, const int experts, const int k, const int n)
{
    if (rows < 32 || !tiles_take(k) || n == 0) return 1;
    const long long there = (long long)std::max(slots / rows, std::min(slots, experts)) * ((n + 255ll) / 256), room = rows == 64 && slots >= 48ll * experts ? 512 : 256;
    return (int)std::max(1ll, std::min({room / there, (long long)(k / 1024), 8ll}));
}

// Workgroups of 256 threads for n columns, `each` to a thread.
static unsigned blocks_across(const int n, const int each) { return (unsigned)((n / each + 255ll) / 256); }

// K in so many parts, of whole quads of steps.
static int cut(ExpertsArgs &p, const int splits)
{
    const int quads = (p.K + 127) / 128, each = (quads + splits - 1) / splits;
    p.steps_each = 2 * each;
    return p.splits = (quads + each - 1) / each;
}

// The workspace of one product: x made ready, the sums of parts of K, in front of the lists.
struct ProductPlan {
    size_t part;
    int splits;
    ExpertsPlan sorted;
};
static ProductPlan product_plan(const qm_expert_weights *w, const int tokens, const int top_k)
{
    const size_t slots = (size_t)tokens * top_k;
    const auto lists = [&](const size_t at) { return experts_plan(false, tokens, top_k, w->experts, (int)((w->n + 255ll) / 256), w->k, w->group, at); };
    ProductPlan p{};
    p.part = ready_bytes(slots, w->k);
    p.splits = splits_of(lists(0).rows, tokens * top_k, w->experts, w->k, w->n);
    p.sorted = lists(p.part + (p.splits > 1 ? up256(p.splits * slots * w->n * 4) : 0));
    return p;
}

// The workspace of the gated MLP: the gated products, x and they made ready, the outputs of the experts, in front of the lists.
struct MlpPlan {
    size_t x_ready, hidden_ready, part;
    int splits;  // of K, where the second product is in tiles
    ExpertsPlan sorted;
};
static MlpPlan mlp_plan(const int tokens, const int top_k, const qm_expert_weights *up, const qm_expert_weights *down)
{
    const int experts = up->experts, inner = down->k, hidden = down->n;
    const auto lists = [&](const size_t at) { return experts_plan(true, tokens, top_k, experts, (int)((inner + 127ll) / 128), hidden, up->group, at); };
    const size_t slots = (size_t)tokens * top_k;
    MlpPlan p{};
    p.x_ready = up256(slots * (tiles_take(inner) ? ready_stride(inner) : inner) * 2);
    p.hidden_ready = p.x_ready + ready_bytes(tokens, hidden);
    p.part = p.hidden_ready + ready_bytes(slots, inner);
    p.splits = splits_of(lists(0).rows, tokens * top_k, experts, inner, hidden);
    p.sorted = lists(p.part + up256(p.splits * slots * hidden * 4));
    return p;
}

}  // namespace qm

using namespace qm;

QM_EXPORT int qm_moe_route(const void *logits, int dtype, long long row_stride, int tokens, int experts, int top_k, const float *bias, int scores, int groups, int top_groups,
                           int group_best, int renormalise, double scale, int *chosen, float *weights, void *stream)
{
    if (dtype != QM_IN_F16 && dtype != QM_IN_BF16 && dtype != QM_IN_F32) return QM_ERR_DTYPE;
    if (tokens < 0 || experts < 1 || experts > QM_ROUTE_EXPERTS || groups < 1 || groups > 64 || experts % groups != 0 || top_groups < 1 || top_groups > groups) return QM_ERR_SHAPE;
    if (top_k < 1 || top_k > 64 || top_k > experts / groups * top_groups || (tokens > 1 && row_stride < experts)) return QM_ERR_SHAPE;
    if ((scores != QM_SCORES_SOFTMAX && scores != QM_SCORES_SIGMOID) || (group_best != 1 && group_best != 2)) return QM_ERR_SHAPE;
    if (tokens == 0) return QM_OK;
    if (!logits || !chosen || !weights) return QM_ERR_NULL;
    if (((uintptr_t)logits & (dtype == QM_IN_F32 ? 3 : 1)) || (((uintptr_t)bias | (uintptr_t)chosen | (uintptr_t)weights) & 3)) return QM_ERR_ALIGN;
    // 16 lanes to a token where so many tokens keep the chip busy all the same, else 64. us with 64 and 16 lanes, bf16: softmax, 8 of 128: 1024 tokens 4.9, 4.8; 2048 5.0, 4.8;
    // 16384 14.1, 7.3; of 256: 1024 5.3, 6.1; 4096 6.8, 6.1; 16384 16.8, 10.6. Sigmoid, 8 of 256 in 4 of 8 groups: 4096 12.3, 14.8; 8192 20.1, 17.5; 65536 131, 119.
    const bool by_logits = scores == QM_SCORES_SOFTMAX && !bias && top_groups == groups;
    const bool narrow = tokens > (by_logits && experts <= 128 ? 1024 : 4096) && experts <= 256 && top_k <= 16 && groups <= 16;
    int parts = 1;
    while (parts * 2 * groups <= (narrow ? 16 : 64)) parts *= 2;
    const RouteArgs p{logits, bias, chosen, weights, tokens > 1 ? row_stride : experts, tokens, experts, top_k, groups, top_groups, scores == QM_SCORES_SIGMOID, group_best == 2,
                      renormalise != 0, parts, (uint32_t)(((1 << 20) + experts / groups - 1) / (experts / groups)), scale};
    const auto run = [&](auto t, auto l) {
        constexpr int T = decltype(t)::value;
        constexpr bool LOGITS = decltype(l)::value;
        const auto kernel = narrow ? experts <= 64    ? &route_kernel<T, 4, 16, LOGITS>
                                     : experts <= 128 ? &route_kernel<T, 8, 16, LOGITS>
                                                      : &route_kernel<T, 16, 16, LOGITS>
                            : experts <= 64    ? &route_kernel<T, 1, 64, LOGITS>
                            : experts <= 128   ? &route_kernel<T, 2, 64, LOGITS>
                            : experts <= 256   ? &route_kernel<T, 4, 64, LOGITS>
                                               : &route_kernel<T, 16, 64, LOGITS>;
        const int each = narrow ? 16 : 4;
        return enqueue(kernel, dim3((unsigned)std::min(((long long)tokens + each - 1) / each, 1ll << 20)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), p);
    };
    const auto by_type = [&](auto t) { return by_logits ? run(t, std::true_type{}) : run(t, std::false_type{}); };
    const hipError_t e = dtype == QM_IN_F16    ? by_type(std::integral_constant<int, QM_IN_F16>{})
                         : dtype == QM_IN_BF16 ? by_type(std::integral_constant<int, QM_IN_BF16>{})
                                               : by_type(std::integral_constant<int, QM_IN_F32>{});
    return e == hipSuccess ? QM_OK : fail_launch(e);
}

// what both products check of tokens and choices; their kernels go through these by eights and sixty-fours in an int
static int check_choices(const int tokens, const int top_k, const int dtype)
{
    if (dtype != QM_IN_F16 && dtype != QM_IN_BF16) return QM_ERR_DTYPE;
    return tokens < 0 || top_k < 0 || (long long)tokens * top_k > INT_MAX - 63 ? QM_ERR_SHAPE : QM_OK;
}

QM_EXPORT size_t qm_gemm_experts_workspace_bytes(const qm_expert_weights *weights, int tokens, int top_k)
{
    if (check_sizes(weights, weights ? weights->scale_dtype : 0) != QM_OK || check_choices(tokens, top_k, QM_IN_F16) != QM_OK) return 0;
    return product_plan(weights, tokens, top_k).sorted.bytes;
}

QM_EXPORT int qm_gemm_experts_i4(const void *x, int dtype, long long token_stride, long long choice_stride, const int *chosen, const qm_expert_weights *weights, void *y,
                                 int tokens, int top_k, void *stream, void *workspace, size_t workspace_bytes)
{
    if (const int e = check_choices(tokens, top_k, dtype); e != QM_OK) return e;
    if (const int e = check_weights(weights, dtype); e != QM_OK) return e;
    if (token_stride < 0 || choice_stride < 0) return QM_ERR_SHAPE;
    if (tokens == 0 || top_k == 0 || weights->n == 0) return QM_OK;
    if (!chosen || !y || (!x && weights->k > 0)) return QM_ERR_NULL;
    if ((((uintptr_t)x | (uintptr_t)y) & 1) || ((uintptr_t)chosen & 3) || ((uintptr_t)workspace & 15)) return QM_ERR_ALIGN;
    const ProductPlan product = product_plan(weights, tokens, top_k);
    const ExpertsPlan &plan = product.sorted;
    if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes)) return QM_ERR_SCRATCH;
    char *const at = static_cast<char *>(workspace);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    ExpertsArgs p = args_of(weights, x, token_stride, choice_stride, chosen, y, tokens, top_k, plan, at);
    const ExpertsKernel kernel = kernel_of(p, plan);
    const ExpertsReady ready = kernel == EXPERTS_TILES ? make_ready(p, dtype, at) : ExpertsReady{};
    hipError_t e = sorts(kernel, p.slots) ? sort_slots(plan, chosen, p.slots, p.experts, ready, dtype, at, s) : hipSuccess;
    if (kernel != EXPERTS_TILES || product.splits == 1) {
        if (e == hipSuccess) e = launch_product(p, kernel, plan, dtype, weights->scale_dtype, EXPERTS_PLAIN, s);
        return e == hipSuccess ? QM_OK : fail_launch(e);
    }
    const int splits = cut(p, product.splits);
    float *const part = reinterpret_cast<float *>(at + product.part);
    p.out = part;
    if (e == hipSuccess) e = launch_product(p, kernel, plan, dtype, weights->scale_dtype, EXPERTS_PART, s);
    if (e == hipSuccess) {
        const bool fours = p.N % 4 == 0;
        const auto join = dtype == QM_IN_F16 ? fours ? &experts_join_kernel<QM_IN_F16, 4> : &experts_join_kernel<QM_IN_F16, 1> : fours ? &experts_join_kernel<QM_IN_BF16, 4> : &experts_join_kernel<QM_IN_BF16, 1>;
        e = enqueue(join, dim3(blocks_across(p.N, fours ? 4 : 1), std::min(p.slots, 65535)), dim3(256), 0, s, part, splits, chosen, p.bias, static_cast<uint16_t *>(y), p.slots, p.experts, p.N);
    }
    return e == hipSuccess ? QM_OK : fail_launch(e);
}

static int check_mlp_sizes(const qm_expert_weights *up, const qm_expert_weights *down, const int dtype)
{
    if (const int e = check_sizes(up, dtype); e != QM_OK) return e;
    if (const int e = check_sizes(down, dtype); e != QM_OK) return e;
    return (long long)down->k * 2 != up->n || down->n != up->k || up->experts != down->experts || up->bias || down->bias ? QM_ERR_SHAPE : QM_OK;
}

QM_EXPORT size_t qm_moe_mlp_workspace_bytes(const qm_expert_weights *up, const qm_expert_weights *down, int tokens, int top_k)
{
    if (!up || !down || check_mlp_sizes(up, down, up->scale_dtype == QM_IN_F32 ? down->scale_dtype : up->scale_dtype) != QM_OK || check_choices(tokens, top_k, QM_IN_F16) != QM_OK) return 0;
    return mlp_plan(tokens, top_k, up, down).sorted.bytes;
}

QM_EXPORT int qm_moe_mlp_i4(const void *x, int dtype, long long token_stride, const int *chosen, const float *weights, const qm_expert_weights *up, const qm_expert_weights *down,
                            void *y, int tokens, int top_k, void *stream, void *workspace, size_t workspace_bytes)
{
    if (const int e = check_choices(tokens, top_k, dtype); e != QM_OK) return e;
    if (const int e = check_weights(up, dtype); e != QM_OK) return e;
    if (const int e = check_weights(down, dtype); e != QM_OK) return e;
    if (const int e = check_mlp_sizes(up, down, dtype); e != QM_OK) return e;
    if (token_stride < 0) return QM_ERR_SHAPE;
    if (tokens == 0 || down->n == 0) return QM_OK;
    if (!y || !x || (top_k > 0 && (!chosen || !weights))) return QM_ERR_NULL;
    if ((((uintptr_t)x | (uintptr_t)y) & 1) || (((uintptr_t)chosen | (uintptr_t)weights) & 3) || ((uintptr_t)workspace & 15)) return QM_ERR_ALIGN;
    const MlpPlan plan = mlp_plan(tokens, top_k, up, down);
    if (plan.sorted.bytes > 0 && (!workspace || workspace_bytes < plan.sorted.bytes)) return QM_ERR_SCRATCH;
    char *const at = static_cast<char *>(workspace);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipError_t e = hipSuccess;
    int splits = 1;
    if (top_k > 0) {
        ExpertsArgs first = args_of(up, x, token_stride, 0, chosen, at, tokens, top_k, plan.sorted, at);
        ExpertsArgs second = args_of(down, at, (long long)top_k * down->k, down->k, chosen, at + plan.part, tokens, top_k, plan.sorted, at);
        const ExpertsKernel one = kernel_of(first, plan.sorted), two = kernel_of(second, plan.sorted);
        splits = two == EXPERTS_TILES ? cut(second, plan.splits) : 1;
        // A token's choices one after the other, added up on the way: one launch less, but weights that two tokens share are read twice. us, experts by themselves and added up
        // on the way, 8 of 128 of 2048 x 1024: 4 tokens 28.6, 25.9; 8 35.1, 33.6; 9 40.2, 43.5; of 256: 8 38.6, 36.0; 9 45.6, 46.6; 16 60.2, 63.9; 2 of 8 of 4096 x 14336: 1 token
        // 36.2, 34.4; 3 71.6, 85.0; 6 of 64 of 2048 x 1408: 4 29.8, 28.3; 6 36.3, 37.5.
        const bool apart = two == EXPERTS_ROWS && (tokens == 1 || (first.slots <= 64 && first.slots * 2 <= up->experts));
        const ExpertsReady ready = one == EXPERTS_TILES ? make_ready(first, dtype, at + plan.x_ready) : ExpertsReady{};
        if (sorts(one, first.slots) || (!apart && sorts(two, first.slots))) e = sort_slots(plan.sorted, chosen, first.slots, up->experts, ready, dtype, at, s);
        // (float16 products are left as the second one's tiles want them; others they make ready first)
        first.pairs_out = one == EXPERTS_TILES && two == EXPERTS_TILES && dtype == QM_IN_F16;
        if (e == hipSuccess && down->k > 0) e = launch_product(first, one, plan.sorted, dtype, up->scale_dtype, EXPERTS_GATED, s);
        if (first.pairs_out) {
            second.ready = reinterpret_cast<const uint16_t *>(at), second.shared = 0;
        } else if (two == EXPERTS_TILES && e == hipSuccess) {
            const ExpertsReady again = make_ready(second, dtype, at + plan.hidden_ready);
            e = sort_slots(plan.sorted, chosen, 0, 0, again, dtype, at, s);
        }
        if (apart) {
            second.out = y, second.shares = weights;
            if (e == hipSuccess) e = launch_product(second, two, plan.sorted, dtype, down->scale_dtype, EXPERTS_SUM, s);
            return e == hipSuccess ? QM_OK : fail_launch(e);
        }
        if (e == hipSuccess) e = launch_product(second, two, plan.sorted, dtype, down->scale_dtype, EXPERTS_PART, s);
    }
    if (e == hipSuccess) {
        const float *const part = reinterpret_cast<const float *>(at + plan.part);
        const bool fours = down->n % 4 == 0;
        const auto sum = dtype == QM_IN_F16 ? fours ? &experts_sum_kernel<QM_IN_F16, 4> : &experts_sum_kernel<QM_IN_F16, 1> : fours ? &experts_sum_kernel<QM_IN_BF16, 4> : &experts_sum_kernel<QM_IN_BF16, 1>;
        e = enqueue(sum, dim3(blocks_across(down->n, fours ? 4 : 1), std::min(tokens, 65535)), dim3(256), 0, s, part, splits, chosen, weights, static_cast<uint16_t *>(y), tokens, top_k, up->experts, down->n);
    }
    return e == hipSuccess ? QM_OK : fail_launch(e);
}
