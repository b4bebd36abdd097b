// The kernels of experts' products on one type of activations (QM_EXPERTS_TYPE: QM_IN_F16 or QM_IN_BF16), and which of them runs.
#include <algorithm>

#include "qm_launch.hpp"
#include "qm_experts_tile.hpp"

namespace qm {

template <int T, int S, ExpertsOut OUT>
static hipError_t launch_any(const ExpertsArgs &p, hipStream_t s)
{
    const int columns = OUT == EXPERTS_GATED ? p.N / 2 : p.N;
    return enqueue(&experts_any_kernel<T, S, OUT>, dim3(std::min(columns / 4 + 1, 1 << 20), std::min(p.slots, 65535)), dim3(256), 0, s, p);
}
template <int T, int S, int G, ExpertsOut OUT>
static hipError_t launch_rows(const ExpertsArgs &p, const ExpertsPlan &plan, hipStream_t s)
{
    const int columns = OUT == EXPERTS_GATED ? p.N / 2 : p.N;
    const auto rows = [&](auto r, auto c, auto nw) {
        constexpr int R = decltype(r)::value, C = decltype(c)::value, NW = decltype(nw)::value;
        typedef ExpertsRowsShape<G, R, C, NW, OUT> Shape;
        static std::atomic<bool> known[QM_MAX_DEVICES] = {};
        const auto kernel = &experts_rows_kernel<T, S, G, R, C, NW, OUT>;
        if (const hipError_t e = ensure_dynamic_lds(kernel, Shape::BYTES, known); e != hipSuccess) return e;
        const long long items = (long long)(OUT == EXPERTS_SUM ? p.slots / p.top_k : plan.tiles) * ((columns + Shape::COLUMNS - 1) / Shape::COLUMNS);
        return enqueue(kernel, dim3((unsigned)std::min<long long>(items, 256 * Shape::PER_CU)), dim3(64 * NW), Shape::BYTES, s, p);
    };
    // Eight waves to an item where there are no more items than CUs and each is long: us with four and eight, a token's product with 2 of 8 experts, N 4096 (256 items): K 2048
    // 5.2, 5.2; 4096 6.8, 6.4; 14336 16.2, 13.0; with 3 of them (384 items): 14336 19.9, 20.2.
    const std::integral_constant<int, 1> i1{};
    const std::integral_constant<int, 2> i2{};
    const std::integral_constant<int, 4> i4{};
    const std::integral_constant<int, 8> i8{};
    const std::integral_constant<int, 16> i16{};
    const bool eight = (long long)std::min(p.slots, p.experts) * ((columns + 31) / 32) <= 256 && p.K >= 4096;
    // (a token's choices one after the other: as many waves as a workgroup can have, and items of 16 columns where those of 32 are for half of the CUs: us of the MLP with 32
    // and 16, 2 tokens, 8 of 128 of 2048 x 1024 (128 items of 32): 17.7, 16.6; 3 (192): 22.5, 24.2; 1 of 2 of 8 of 4096 x 14336 (128): 38.7, 34.3; 2 (256): 68.8, 72.0)
    if constexpr (OUT == EXPERTS_SUM) return (long long)(p.slots / p.top_k) * ((columns + 31) / 32) <= 128 ? rows(i2, i1, i16) : rows(i2, i2, i16);
    else switch (plan.rows) {
    case 2: return eight ? rows(i2, i2, i8) : rows(i2, i2, i4);
    case 4: return eight ? rows(i4, i2, i8) : rows(i4, i2, i4);
    case 8: return eight ? rows(i8, i2, i8) : rows(i8, i2, i4);
    default: return eight ? rows(i16, i2, i8) : rows(i16, i2, i4);
    }
}
template <int T, int S, int G, ExpertsOut OUT>
static hipError_t launch_tiles(const ExpertsArgs &p, const ExpertsPlan &plan, hipStream_t s)
{
    const int columns = OUT == EXPERTS_GATED ? p.N / 2 : p.N;
    const auto tiles = [&](auto mt) {
        typedef ExpertsTileShape<G, decltype(mt)::value, OUT> Shape;
        static std::atomic<bool> known[QM_MAX_DEVICES] = {};
        const auto kernel = &experts_tile_kernel<T, S, G, decltype(mt)::value, OUT>;
        if (const hipError_t e = ensure_dynamic_lds(kernel, Shape::BYTES, known); e != hipSuccess) return e;
        return enqueue(kernel, dim3(plan.tiles * Shape::across(columns) * (OUT == EXPERTS_PART ? p.splits : 1)), dim3(Shape::THREADS), Shape::BYTES, s, p);
    };
    return plan.rows == 64 ? tiles(std::integral_constant<int, 2>{}) : tiles(std::integral_constant<int, 1>{});
}

#if QM_EXPERTS_TYPE == QM_IN_F16
#define QM_LAUNCH_EXPERTS launch_experts_f16
#else
#define QM_LAUNCH_EXPERTS launch_experts_bf16
#endif
hipError_t QM_LAUNCH_EXPERTS(const ExpertsArgs &p, const ExpertsPlan &plan, const int scale_dtype, const ExpertsOut out, const ExpertsKernel kernel, hipStream_t s)
{
    constexpr int T = QM_EXPERTS_TYPE;
    const auto by_out = [&](auto st, auto o) {
        constexpr int S = decltype(st)::value;
        constexpr ExpertsOut OUT = (ExpertsOut)decltype(o)::value;
        if (kernel == EXPERTS_ROWS) return p.group % 128 == 0 ? launch_rows<T, S, 4, OUT>(p, plan, s) : p.group % 64 == 0 ? launch_rows<T, S, 2, OUT>(p, plan, s) : launch_rows<T, S, 1, OUT>(p, plan, s);
        if constexpr (OUT == EXPERTS_SUM) return hipErrorInvalidValue;  // (no other kernel adds up)
        else if (kernel == EXPERTS_ANY) return launch_any<T, S, OUT>(p, s);
        else return p.group % 128 == 0 ? launch_tiles<T, S, 4, OUT>(p, plan, s) : p.group % 64 == 0 ? launch_tiles<T, S, 2, OUT>(p, plan, s) : launch_tiles<T, S, 1, OUT>(p, plan, s);
    };
    const auto by_type = [&](auto st) {
        switch (out) {
        case EXPERTS_PLAIN: return by_out(st, std::integral_constant<int, EXPERTS_PLAIN>{});
        case EXPERTS_GATED: return by_out(st, std::integral_constant<int, EXPERTS_GATED>{});
        case EXPERTS_PART: return by_out(st, std::integral_constant<int, EXPERTS_PART>{});
        default: return by_out(st, std::integral_constant<int, EXPERTS_SUM>{});
        }
    };
    return scale_dtype == QM_IN_F32 ? by_type(std::integral_constant<int, QM_IN_F32>{}) : by_type(std::integral_constant<int, T>{});
}

}  // namespace qm
