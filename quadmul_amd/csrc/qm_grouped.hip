// C entries of the GEMM on 16-bit activations and int4 weights with group scales (include/qm_abi.h): argument checks,
// choice of kernel, launch.
#include <algorithm>

#include "../../include/qm_abi.h"
#include "qm_launch.hpp"
#include "qm_grouped.hpp"

#define QM_EXPORT extern "C" __attribute__((visibility("default")))

namespace qm {

template <int T, int S, int MODE>
static hipError_t launch_skinny_mode(const GroupedArgs &p, hipStream_t s)
{
    constexpr int NW = 8;
    const auto go = [&](auto kernel, int nt) { return enqueue(kernel, dim3((p.N + 16 * nt - 1) / (16 * nt)), dim3(NW * 64), 0, s, p); };
    if (p.M <= 16) return p.N <= 6144 ? go(&gemm_grouped_skinny_kernel<T, S, MODE, 1, 1, NW>, 1) : go(&gemm_grouped_skinny_kernel<T, S, MODE, 1, 2, NW>, 2);
    if (p.M <= 32) return go(&gemm_grouped_skinny_kernel<T, S, MODE, 2, 2, NW>, 2);
    return go(&gemm_grouped_skinny_kernel<T, S, MODE, 4, 2, NW>, 2);
}
template <int T, int S>
static hipError_t launch_grouped(const GroupedArgs &p, hipStream_t s)
{
    if (p.K > 0 && p.K % 32 == 0 && ((uintptr_t)p.B & 15) == 0 && p.M <= 64) {
        switch (group_mode(p.group)) {
        case 1: return launch_skinny_mode<T, S, 1>(p, s);
        case 2: return launch_skinny_mode<T, S, 2>(p, s);
        case 4: return launch_skinny_mode<T, S, 4>(p, s);
        default: return launch_skinny_mode<T, S, 0>(p, s);
        }
    }
    const int rows = (p.M + GROUPED_ROWS - 1) / GROUPED_ROWS;
    return enqueue(&gemm_grouped_any_kernel<T, S>, dim3((p.N + 3) / 4, std::min(rows, 65535)), dim3(256), 0, s, p);
}

}  // namespace qm

using namespace qm;

QM_EXPORT size_t qm_gemm_grouped_workspace_bytes(int, int, int, int, int) { return 0; }

QM_EXPORT int qm_gemm_grouped_i4(const void *x, int dtype, long long x_stride, const void *B, const void *scale, int scale_dtype, int group,
                                 const void *bias, void *D, int m, int n, int k, void *stream, void *workspace, size_t workspace_bytes)
{
    if (dtype != QM_IN_F16 && dtype != QM_IN_BF16) return QM_ERR_DTYPE;
    if (scale_dtype != QM_IN_F32 && scale_dtype != dtype) return QM_ERR_DTYPE;
    if (m < 0 || n < 0 || k < 0 || (k & 1) || group < 32 || group % 32 != 0 || (m > 1 && x_stride < k)) return QM_ERR_SHAPE;
    if (m == 0 || n == 0) return QM_OK;
    if (!D || (k > 0 && (!x || !B || !scale))) return QM_ERR_NULL;
    if ((((uintptr_t)x | (uintptr_t)D | (uintptr_t)bias) & 1) || ((uintptr_t)scale & (scale_dtype == QM_IN_F32 ? 3 : 1)) || ((uintptr_t)workspace & 15)) return QM_ERR_ALIGN;
    if (workspace_bytes < qm_gemm_grouped_workspace_bytes(m, n, k, group, 0)) return QM_ERR_SCRATCH;
    const GroupedArgs p{static_cast<const uint16_t *>(x), static_cast<const uint8_t *>(B), scale, static_cast<const uint16_t *>(bias),
                        static_cast<uint16_t *>(D), x_stride, m, n, k, group, (int)(((long long)k + group - 1) / group)};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipError_t e;
    if (dtype == QM_IN_F16) e = scale_dtype == QM_IN_F32 ? launch_grouped<QM_IN_F16, QM_IN_F32>(p, s) : launch_grouped<QM_IN_F16, QM_IN_F16>(p, s);
    else e = scale_dtype == QM_IN_F32 ? launch_grouped<QM_IN_BF16, QM_IN_F32>(p, s) : launch_grouped<QM_IN_BF16, QM_IN_BF16>(p, s);
    return e == hipSuccess ? QM_OK : fail_launch(e);
}
