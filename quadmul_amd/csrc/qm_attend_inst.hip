// The attention kernels for one type of queries: QM_ATTEND_TYPE is QM_IN_F16 or QM_IN_BF16.
#include <algorithm>

#include "qm_launch.hpp"
#include "qm_attend.hpp"

namespace qm {

template <int D>
static hipError_t launch(const KvArgs &c, const AttendArgs &a, hipStream_t s)
{
    constexpr int NW = 4;
    const dim3 grid(a.splits * a.tiles, c.kv_heads, std::min(c.sequences, 65535));
    const hipError_t e = enqueue(&kv_attend_kernel<QM_ATTEND_TYPE, D, NW>, grid, dim3(NW * 64), 0, s, c, a);
    if (e != hipSuccess || a.splits == 1) return e;
    const int rows = c.tokens * a.heads;
    return enqueue(&kv_join_kernel<QM_ATTEND_TYPE, D>, dim3(std::min(rows, 1 << 20)), dim3(256), 0, s, a.part, a.out, rows, a.splits);
}

#if QM_ATTEND_TYPE == QM_IN_F16
hipError_t launch_attend_f16(const KvArgs &c, const AttendArgs &a, hipStream_t s)
#else
hipError_t launch_attend_bf16(const KvArgs &c, const AttendArgs &a, hipStream_t s)
#endif
{
    switch (c.dim) {
    case 64: return launch<64>(c, a, s);
    case 96: return launch<96>(c, a, s);
    case 128: return launch<128>(c, a, s);
    case 192: return launch<192>(c, a, s);
    default: return launch<256>(c, a, s);
    }
}

}  // namespace qm
