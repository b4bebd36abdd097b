// Slots sorted by their expert, for the products of qm_experts.hpp.
#pragma once
#include "qm_experts_tile.hpp"

namespace qm {

// The slots by expert, and tiles of up to `rows` of each expert's. One workgroup: counts, their sums, places, all in the LDS. Which place of its expert's a slot gets is
// chance, and no result depends on it: every row of a tile is summed by itself.
// A chain of latencies, 4.5 us for 256 slots, 13 for 8192 with the rows of x (67 MB moved): the tiles are known on the device only, and nothing waits for the host.
// With it the rows of x made ready, by the workgroups after that one (all of them where there are no slots).
template <int T>
__global__ __launch_bounds__(1024) void experts_sort_kernel(const int *chosen, const int slots, const int experts, const int rows, int *order, int *tiles, int *count, const ExpertsReady ready)
{
    const int sorting = slots > 0 ? 1 : 0;
    if ((int)blockIdx.x >= sorting) {
        experts_ready_rows<T>(ready, ((long long)blockIdx.x - sorting) * 16 + (threadIdx.x >> 6), ((long long)gridDim.x - sorting) * 16);
        return;
    }
    extern __shared__ int bins[];  // [experts + 1]
    __shared__ int sums[2][16];
    constexpr int AHEAD = 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i <= experts; i += 1024) bins[i] = 0;
    __syncthreads();
    const auto for_slots = [&](const auto &use) {
        for (long long from = tid; from < slots; from += 1024 * AHEAD) {
            int e[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) e[i] = chosen[min(from + 1024 * i, (long long)slots - 1)];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (from + 1024 * i < slots) use((int)(from + 1024 * i), (unsigned)e[i] < (unsigned)experts ? e[i] : experts);
        }
    };
    for_slots([&](int, const int bin) { atomicAdd(&bins[bin], 1); });
    __syncthreads();
    const int each = (experts + 1024) / 1024, first = min(tid * each, experts + 1), last = min(first + each, experts + 1);
    int held = 0, made = 0;  // slots and tiles in front of this thread's bins
    for (int b = first; b < last; ++b) held += bins[b], made += (bins[b] + rows - 1) / rows;
    const int my_held = held, my_made = made;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int a = __shfl_up(held, d), b = __shfl_up(made, d);
        if (lane >= d) held += a, made += b;
    }
    if (lane == 63) sums[0][wave] = held, sums[1][wave] = made;
    __syncthreads();
    for (int w = 0; w < wave; ++w) held += sums[0][w], made += sums[1][w];
    if (tid == 1023) count[0] = made;
    held -= my_held, made -= my_made;
    for (int b = first; b < last; ++b) {
        const int n = bins[b];
        if (b == experts) count[1] = made, count[2] = held;
        bins[b] = held;
        for (int i = 0; i < n; i += rows, ++made) *reinterpret_cast<v4i *>(tiles + 4 * (size_t)made) = v4i{b, held + i, min(n - i, rows), 0};
        held += n;
    }
    __syncthreads();
    for_slots([&](const int slot, const int bin) { order[atomicAdd(&bins[bin], 1)] = slot; });
}

}  // namespace qm
