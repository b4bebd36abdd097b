// C entries of the GEMM on 16-bit activations and int4 weights with group scales (include/qm_abi.h): argument checks,
// choice of kernel, launch.
#include <algorithm>
#include <atomic>

#include "../../include/qm_abi.h"
#include "qm_launch.hpp"
#include "qm_grouped.hpp"

#define QM_EXPORT extern "C" __attribute__((visibility("default")))

namespace qm {

// Which kernel runs, and what it needs.
enum GroupedKernel { GROUPED_ANY, GROUPED_ROWS16, GROUPED_TILE };
struct GroupedPlan {
    GroupedKernel kernel;
    int waves, ways, chunk, runs;  // of a workgroup, to a tile of columns; blocks of 32 of K in a run, runs
    int rows;                      // of a tile
    size_t bytes;
};
static GroupedPlan grouped_plan(int m, int n, int k, int align)  // (align: of B; x may be anywhere)
{
    GroupedPlan p{GROUPED_ANY, 16, 1, 0, 1, 0, 0};
    // (a wave reaches up to 64 rows of B with offsets of 32 bits)
    if (k == 0 || k % 32 != 0 || align < 16 || k >= 1 << 26) return p;
    if (m > 16 && n > 65535 * 64) return p;  // (the grid's limit)
    if (m > 16) {
        p.kernel = GROUPED_TILE;
        const int quads = (k / 32 + 3) / 4;
        const auto tiles_of = [&](const int rows) { return (long long)((m + rows - 1) / rows) * ((n + 127) / 128); };
        // 256 rows where that leaves a tile to a CU and no more rows without anything to do than an eighth. By 256 and by 128, us: 900 x 8192 x 8192 147 and
        // 168, 4000 x 28672 x 4096 1034 and 1139, 2048 x 11008 x 4096 222 and 239; with more rows empty, in groups of 32, 300 x 28672 x 4096 223 and 178.
        // (Least sure where an eleventh is empty: 1300 x 11008 x 4096 202 and 169, 1300 x 65536 x 2048 465 and 487.)
        const bool few_empty = (m + 255) / 256 * 2 == (m + 127) / 128 || m >= 1024;
        p.rows = m <= 32 ? 32 : m <= 64 ? 64 : tiles_of(256) >= 256 && few_empty ? 256 : 128;
        // A workgroup to a CU at least, of 1024 elements of K or more. Above 64 rows with groups below 128 tiles have 64 columns: counted as 128 all the same,
        // for two of them to a CU pay for the partial sums: in groups of 32, so and with 64, us, 80 x 11008 x 4096 39 and 50, 256 x 4096 x 11008 53 and 73, 384 x 8192 x
        // 8192 117 and 119, 200 x 28672 x 4096 122 and 116.
        const long long tiles = tiles_of(p.rows);
        p.runs = (int)std::max<long long>(1, std::min<long long>(256 / tiles, quads / 8));
        p.chunk = (quads + p.runs - 1) / p.runs * 4;
        p.runs = (k / 32 + p.chunk - 1) / p.chunk;
        if (p.runs > 1) p.bytes = (size_t)p.runs * m * n * sizeof(float);
        return p;
    }
    p.kernel = GROUPED_ROWS16;
    // what a workgroup holds of x: 128 KiB, beside the sums; one workgroup to a CU
    const int blocks = k / 32, most = (128 << 10) / (64 * (m | 1) + 64) / 8 * 8;
    p.runs = (blocks + most - 1) / most;
    p.chunk = ((blocks + p.runs - 1) / p.runs + 3) / 4 * 4;
    p.runs = (blocks + p.chunk - 1) / p.chunk;
    if (p.runs > 1) p.bytes = (size_t)p.runs * m * n * sizeof(float);
    // Waves enough for the chip. A call that is over before they are all at work has eight to a workgroup: 1 x 4096 x 4096 5.8 us, with sixteen
    // 7.1; 1 x 28672 x 4096 (groups of 32) 20.3 and 20.4, 13 x 8192 x 28672 42 and 39, the two layers of 8 x 4096 x 4096 and 8 x 6144 x 4096 21 and 18.
    const long long tiles = (long long)((n + 15) / 16) * p.runs;
    if (m <= 4 && tiles <= 512) p.waves = 8;
    while (p.ways < p.waves && tiles * p.ways < 3072) p.ways *= 2;
    return p;
}

template <int T, int S, int MODE>
static hipError_t launch_mode(GroupedArgs p, const GroupedPlan &plan, hipStream_t s)
{
    p.chunk = plan.chunk, p.ways = plan.ways;
    if (plan.kernel == GROUPED_TILE) {
        const dim3 grid((p.M + plan.rows - 1) / plan.rows, (p.N + 127) / 128, plan.runs);
        // (with a scale to every one or two blocks the registers of 64 columns to a wave do not fit)
        constexpr int NT = MODE == 1 ? 4 : 2, BN = 32 * NT;
        const auto wide = [&](auto kernel, std::atomic<bool> *known) {
            const int lds = 2 * 8 * 16 * (plan.rows + BN) + 2 * 2 * BN * (int)sizeof(float);
            if (const hipError_t e = ensure_dynamic_lds(kernel, lds, known); e != hipSuccess) return e;
            return enqueue(kernel, dim3(grid.x, (p.N + BN - 1) / BN, grid.z), dim3(plan.rows * 2), lds, s, p);
        };
        static std::atomic<bool> known_wide[2][QM_MAX_DEVICES] = {};
        switch (plan.rows) {
        case 256: return wide(&gemm_grouped_wide_kernel<T, S, MODE, 4, 2, 4, NT>, known_wide[0]);
        case 128: return wide(&gemm_grouped_wide_kernel<T, S, MODE, 2, 2, 4, NT>, known_wide[1]);
        case 64: return enqueue(&gemm_grouped_tile_kernel<T, S, MODE, 4, 2>, grid, dim3(256), 0, s, p);
        case 32: return enqueue(&gemm_grouped_tile_kernel<T, S, MODE, 2, 2>, grid, dim3(256), 0, s, p);
        }
    }
    const int tiles = plan.waves / plan.ways, groups = ((p.N + 15) / 16 + tiles - 1) / tiles;
    const size_t lds = (size_t)plan.chunk * (64 * (p.M | 1) + 64);
    static std::atomic<bool> known[2][QM_MAX_DEVICES] = {};
    const auto kernel = plan.waves == 8 ? &gemm_grouped_rows_kernel<T, S, MODE, 8> : &gemm_grouped_rows_kernel<T, S, MODE, 16>;
    if (const hipError_t e = ensure_dynamic_lds(kernel, 128 << 10, known[plan.waves == 8]); e != hipSuccess) return e;
    return enqueue(kernel, dim3(std::min(groups, std::max(1, 256 / plan.runs)), plan.runs), dim3(plan.waves * 64), lds, s, p);
}
template <int T, int S>
static hipError_t launch_grouped(GroupedArgs p, const GroupedPlan &plan, hipStream_t s)
{
    if (plan.kernel == GROUPED_ANY) {
        const int rows = (p.M + GROUPED_ROWS - 1) / GROUPED_ROWS;
        return enqueue(&gemm_grouped_any_kernel<T, S>, dim3(std::min((unsigned)p.N / 4 + 1, 1u << 22), std::min(rows, 65535)), dim3(256), 0, s, p);
    }
    hipError_t e;
    switch (group_mode(p.group)) {
    case 1: e = launch_mode<T, S, 1>(p, plan, s); break;
    case 2: e = launch_mode<T, S, 2>(p, plan, s); break;
    case 4: e = launch_mode<T, S, 4>(p, plan, s); break;
    default: e = launch_mode<T, S, 0>(p, plan, s); break;
    }
    if (e != hipSuccess || plan.runs == 1) return e;
    return enqueue(&gemm_grouped_join_kernel<T>, dim3((unsigned)std::min<size_t>(((size_t)p.M * p.N + 255) / 256, 4096)), dim3(256), 0, s, p, plan.runs);
}

}  // namespace qm

using namespace qm;

QM_EXPORT size_t qm_gemm_grouped_workspace_bytes(int m, int n, int k, int group, int align)
{
    if (m <= 0 || n <= 0 || k <= 0 || (k & 1) || group < 32 || group % 32 != 0) return 0;
    return grouped_plan(m, n, k, align).bytes;
}

QM_EXPORT int qm_gemm_grouped_i4(const void *x, int dtype, long long x_stride, const void *B, const void *scale, int scale_dtype, int group,
                                 const void *bias, void *D, int m, int n, int k, void *stream, void *workspace, size_t workspace_bytes)
{
    if (dtype != QM_IN_F16 && dtype != QM_IN_BF16) return QM_ERR_DTYPE;
    if (scale_dtype != QM_IN_F32 && scale_dtype != dtype) return QM_ERR_DTYPE;
    if (m < 0 || n < 0 || k < 0 || (k & 1) || group < 32 || group % 32 != 0 || (m > 1 && x_stride < k)) return QM_ERR_SHAPE;
    if (m == 0 || n == 0) return QM_OK;
    if (!D || (k > 0 && (!x || !B || !scale))) return QM_ERR_NULL;
    if ((((uintptr_t)x | (uintptr_t)D | (uintptr_t)bias) & 1) || ((uintptr_t)scale & (scale_dtype == QM_IN_F32 ? 3 : 1)) || ((uintptr_t)workspace & 15)) return QM_ERR_ALIGN;
    const GroupedPlan plan = grouped_plan(m, n, k, ((uintptr_t)B & 15) == 0 ? 16 : 1);
    if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes)) return QM_ERR_SCRATCH;
    const GroupedArgs p{static_cast<const uint16_t *>(x), static_cast<const uint8_t *>(B), scale, static_cast<const uint16_t *>(bias),
                        static_cast<uint16_t *>(D), m > 1 ? x_stride : k, m, n, k, group, (int)(((long long)k + group - 1) / group), 1, 0,
                        plan.bytes > 0 ? static_cast<float *>(workspace) : nullptr};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipError_t e;
    if (dtype == QM_IN_F16) e = scale_dtype == QM_IN_F32 ? launch_grouped<QM_IN_F16, QM_IN_F32>(p, plan, s) : launch_grouped<QM_IN_F16, QM_IN_F16>(p, plan, s);
    else e = scale_dtype == QM_IN_F32 ? launch_grouped<QM_IN_BF16, QM_IN_F32>(p, plan, s) : launch_grouped<QM_IN_BF16, QM_IN_BF16>(p, plan, s);
    return e == hipSuccess ? QM_OK : fail_launch(e);
}
