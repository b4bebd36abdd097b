// The attention kernels for one type of queries: QM_ATTEND_TYPE is QM_IN_F16 or QM_IN_BF16.
#include <algorithm>
#include <atomic>

#include "qm_launch.hpp"
#include "qm_attend.hpp"

namespace qm {

template <int D>
static hipError_t launch(const KvArgs &c, const AttendArgs &a, hipStream_t s)
{
    if (a.wide) {
        constexpr int LDS = (4 * (D / 32) + 2 * (D / 16)) * 64 * 16;  // keys and values of a step
        static std::atomic<bool> known[2][QM_MAX_DEVICES] = {};
        const auto kernel = a.wide == 1 ? &kv_attend_rows_kernel<QM_ATTEND_TYPE, D, 1> : &kv_attend_rows_kernel<QM_ATTEND_TYPE, D, 2>;
        if (const hipError_t e = ensure_dynamic_lds(kernel, a.wide * LDS, known[a.wide - 1]); e != hipSuccess) return e;
        return enqueue(kernel, dim3(a.tiles, std::max(1, std::min(c.sequences, 65535 / c.kv_heads)) * c.kv_heads), dim3(256 * a.wide), a.wide * LDS, s, c, a);
    }
    constexpr int NW = D > 128 ? 4 : 8;  // (with eight the registers of the wider heads do not fit)
    // (up to 2^22 workgroups along a side, of 512 threads: a grid has less than 2^32)
    if (a.parts == 0) return enqueue(&kv_attend_kernel<QM_ATTEND_TYPE, D, NW, false>, dim3(std::min(c.sequences, (1 << 22) / c.kv_heads) * c.kv_heads, a.tiles), dim3(NW * 64), 0, s, c, a);
    const hipError_t e = enqueue(&kv_attend_kernel<QM_ATTEND_TYPE, D, 4, true>, dim3(a.parts * c.kv_heads, a.tiles), dim3(256), 0, s, c, a);
    if (e != hipSuccess) return e;
    return enqueue(&kv_join_kernel<QM_ATTEND_TYPE, D, 8>, dim3(a.rows, a.tiles * c.kv_heads, c.sequences), dim3(512), 0, s, c, a);
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
