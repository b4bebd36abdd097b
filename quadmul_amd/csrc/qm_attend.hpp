// Attention over the paged 8-bit cache (qm_kv.hpp).
#pragma once
#include "qm_kv.hpp"

namespace qm {

struct AttendArgs {
    const uint16_t *q;
    uint16_t *out;
    long long q_token, q_head;
    int heads, causal, window;
    float scale;
};

// A workgroup to a query token (blockIdx.x) and a head (blockIdx.y): 256 tokens of the cache at a time, a thread to a token for the
// scores and a thread to a channel for the sum of the values.
template <int T>
__global__ __launch_bounds__(256) void kv_attend_kernel(const KvArgs c, const AttendArgs a)
{
    __shared__ float query[256], weight[256], part[4];
    const int tid = threadIdx.x, head = blockIdx.y, kv_head = head / (a.heads / c.kv_heads);
    for (int row = blockIdx.x; row < c.tokens; row += gridDim.x) {
        int s = 0;
        if (c.start == nullptr) {
            s = row / c.per;
        } else {
            for (int lo = 0, hi = c.sequences; lo < hi;) {  // the last sequence that begins at or before the row
                const int mid = (lo + hi) / 2;
                if (c.start[mid] <= row) s = mid, lo = mid + 1;
                else hi = mid;
            }
        }
        const KvSequence q = kv_sequence(c, s);
        const int position = q.begin + row - q.row0;
        const bool here = row >= q.row0 && row < q.row0 + q.count && position >= 0;
        const long long most = (long long)c.width * c.page;
        const int end = !here ? 0 : (int)min((long long)(a.causal ? position + 1 : q.length), most);
        const int begin = a.window > 0 ? max(position - a.window + 1, 0) : 0;
        __syncthreads();
        if (tid < c.dim) query[tid] = float_of<T>(a.q[row * a.q_token + head * a.q_head + tid]) * a.scale;
        float top = -INFINITY, total = 0.0f, sum = 0.0f;
        for (int base = begin / 256 * 256; base < end; base += 256) {
            __syncthreads();
            const int token = base + tid;
            const int id = token >= begin && token < end ? kv_page(c, s, token / c.page) : -1;
            float score = -INFINITY, vs = 0.0f;
            if (id >= 0) {
                const size_t at = (size_t)id * c.kv_heads + kv_head;
                const int8_t *const key = c.k + (at * c.page + token % c.page) * c.dim;
                float dot = 0.0f;
                for (int d = 0; d < c.dim; ++d) dot = __builtin_fmaf(query[d], (float)key[d], dot);
                score = dot * c.scales[at * 2];
                vs = c.scales[at * 2 + 1];
            }
            float high = score;
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) high = fmaxf(high, __shfl_xor(high, d));
            if ((tid & 63) == 0) part[tid >> 6] = high;
            __syncthreads();
            high = fmaxf(top, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
            const float finite = high == -INFINITY ? 0.0f : high, p = expf(score - finite), old = expf(top - finite);
            top = high;
            weight[tid] = id >= 0 ? p * vs : 0.0f;
            float all = p;
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) all += __shfl_xor(all, d);
            __syncthreads();
            if ((tid & 63) == 0) part[tid >> 6] = all;
            __syncthreads();
            total = total * old + (part[0] + part[1] + part[2] + part[3]);
            sum *= old;
            if (tid < c.dim) {
                for (int j = 0; j < 256; j += c.page) {
                    const int page = kv_page(c, s, (base + j) / c.page);
                    if (page < 0 || base + j >= end || base + j + c.page <= begin) continue;
                    const int8_t *const values = c.v + (((size_t)page * c.kv_heads + kv_head) * c.dim + tid) * c.page;
                    for (int i = 0; i < c.page; ++i) sum = __builtin_fmaf(weight[j + i], (float)values[i], sum);
                }
            }
        }
        if (tid < c.dim) a.out[((size_t)row * a.heads + head) * c.dim + tid] = round16<T>(total == 0.0f ? 0.0f : sum / total);
    }
}

}  // namespace qm
