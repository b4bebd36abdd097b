// PyTorch-ROCm extension module `quadmul`: the drop-in for the reference's
// pybind11 module (extension.cpp:8-29) -- same module name (setup.py:8,11), same
// function gemm(a, b, c, m, n, k) -> None, same positional order (test.py:40).
// Host-only C++: tensors are unwrapped to device pointers and handed, with the
// current HIP stream of a's device (extension.cpp:23), to the C ABI in
// include/qm_abi.h.  No kernels and no HIP runtime calls live here.
//
// The argument checks the reference left commented out (extension.cpp:11-15) are
// live here; a non-zero status from the library is raised as RuntimeError.
#include <torch/extension.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/Exception.h>

#include "qm_abi.h"

namespace {

void check_status(int status, const char *what)
{
    if (status == QM_OK) return;
    if (status == QM_ERR_LAUNCH)
        TORCH_CHECK(false, what, ": ", qm_status_string(status), " (hipError_t ", qm_last_hip_error(), ")");
    TORCH_CHECK(false, what, ": ", qm_status_string(status));
}

bool is_byte(const torch::Tensor &t) { return t.scalar_type() == torch::kInt8 || t.scalar_type() == torch::kUInt8; }

void *stream_of(const torch::Tensor &t) { return static_cast<void *>(c10::hip::getCurrentHIPStream(t.get_device()).stream()); }

void check_operands(const torch::Tensor &a, const torch::Tensor &b, const torch::Tensor &c, int64_t m, int64_t n, int64_t k,
                    bool scaled = false)
{
    TORCH_CHECK(a.is_cuda() && b.is_cuda() && c.is_cuda(), "quadmul.gemm: a, b and c must be GPU tensors");
    TORCH_CHECK(a.device() == b.device() && a.device() == c.device(), "quadmul.gemm: all tensors must be on the same device");
    // pack_b yields int8 (test.py:14); the reference only ever looks at data_ptr().
    TORCH_CHECK(is_byte(a) && is_byte(b), "quadmul.gemm: a and b must be int8 or uint8 (packed int4)");
    if (scaled) {
        TORCH_CHECK(c.scalar_type() == torch::kFloat16 || c.scalar_type() == torch::kBFloat16, "quadmul.gemm_scaled: d must be float16 or bfloat16");
    } else {
        TORCH_CHECK(c.scalar_type() == torch::kInt32, "quadmul.gemm: c must be int32");
    }
    TORCH_CHECK(a.is_contiguous() && b.is_contiguous() && c.is_contiguous(), "quadmul.gemm: all tensors must be contiguous");
    TORCH_CHECK(m >= 0 && n >= 0 && k >= 0 && k % 2 == 0, "quadmul.gemm: m, n, k must be >= 0 and k even");
    TORCH_CHECK(m <= INT32_MAX && n <= INT32_MAX && k <= INT32_MAX, "quadmul.gemm: m, n, k must fit in int32");
    TORCH_CHECK(a.numel() == m * (k / 2), "quadmul.gemm: a must hold m*k/2 bytes, got ", a.numel());
    TORCH_CHECK(b.numel() == n * (k / 2), "quadmul.gemm: b must hold n*k/2 bytes, got ", b.numel());
    TORCH_CHECK(c.numel() == m * n, "quadmul.gemm: c must hold m*n int32, got ", c.numel());
}

// The workspace of a call that splits K (few output tiles, long K), from torch's caching
// allocator: stream-ordered, so calls on different streams never share one, and legal under
// graph capture.  An undefined tensor when the shape does not split.
int ptr_alignment(const torch::Tensor &a, const torch::Tensor &b)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.data_ptr()) | reinterpret_cast<uintptr_t>(b.data_ptr());
    if (x == 0) return 4096;
    const uintptr_t low = x & (~x + 1);
    return low > 4096 ? 4096 : (int)low;
}

// Bytes that only make a call faster: an undefined tensor where the allocator does not have them, and the call runs
// without (in a capture too: what it asks for there is the graph's pool, and nothing has been enqueued yet).
torch::Tensor bytes_if_there_are(size_t bytes, const torch::TensorOptions &options)
{
    try {
        return torch::empty({(int64_t)bytes}, options.dtype(torch::kUInt8));
    } catch (const c10::OutOfMemoryError &) {
        return torch::Tensor();
    }
}

torch::Tensor workspace_for(const torch::Tensor &a, const torch::Tensor &b, int64_t m, int64_t n, int64_t k, int cfg, bool scaled)
{
    const int align = ptr_alignment(a, b);
    const size_t need = qm_gemm_workspace_bytes((int)m, (int)n, (int)k, align, cfg, scaled ? 1 : 0);
    const size_t faster = cfg == QM_CFG_AUTO ? qm_gemm_recode_bytes((int)m, (int)n, (int)k, align, scaled ? 1 : 0) : 0;
    if (faster > need) {
        const torch::Tensor ws = bytes_if_there_are(faster, a.options());
        if (ws.defined()) return ws;
    }
    if (need == 0) return torch::Tensor();
    return torch::empty({(int64_t)need}, a.options().dtype(torch::kUInt8));
}

void gemm(torch::Tensor a, torch::Tensor b, torch::Tensor c, int64_t m, int64_t n, int64_t k)
{
    check_operands(a, b, c, m, n, k);
    c10::OptionalDeviceGuard guard(a.device());
    const torch::Tensor ws = workspace_for(a, b, m, n, k, QM_CFG_AUTO, false);
    check_status(qm_gemm_i4_ws(a.data_ptr(), b.data_ptr(), c.data_ptr(), (int)m, (int)n, (int)k, stream_of(a), QM_CFG_AUTO,
                               ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (size_t)ws.numel() : 0),
                 "quadmul.gemm");
}

// The GEMM with the dequantising epilogue fused in (no counterpart in the reference's code;
// its README.md:7 names the idea): d = round(((float)c * row_scale[m]) * col_scale[n]), d
// float16 or bfloat16, the scales float32 vectors on a's device (an undefined tensor = ones).
void check_scale(const c10::optional<torch::Tensor> &s, const torch::Tensor &a, int64_t count, const char *what)
{
    if (!s.has_value()) return;
    TORCH_CHECK(s->is_cuda() && s->device() == a.device() && s->scalar_type() == torch::kFloat32 && s->is_contiguous() && s->numel() == count,
                "quadmul.gemm_scaled: ", what, " must be a contiguous float32 vector of ", count, " elements on a's device");
}

void gemm_scaled(torch::Tensor a, torch::Tensor b, torch::Tensor d, int64_t m, int64_t n, int64_t k,
                 c10::optional<torch::Tensor> row_scale, c10::optional<torch::Tensor> col_scale)
{
    check_operands(a, b, d, m, n, k, true);
    check_scale(row_scale, a, m, "row_scale");
    check_scale(col_scale, a, n, "col_scale");
    c10::OptionalDeviceGuard guard(a.device());
    const int out = d.scalar_type() == torch::kFloat16 ? QM_OUT_F16 : QM_OUT_BF16;
    const torch::Tensor ws = workspace_for(a, b, m, n, k, QM_CFG_AUTO, true);
    check_status(qm_gemm_i4_scaled_ws(a.data_ptr(), b.data_ptr(), d.data_ptr(), (int)m, (int)n, (int)k,
                                      row_scale.has_value() ? row_scale->data_ptr<float>() : nullptr,
                                      col_scale.has_value() ? col_scale->data_ptr<float>() : nullptr, out, stream_of(a), QM_CFG_AUTO,
                                      ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (size_t)ws.numel() : 0),
                 "quadmul.gemm_scaled");
}

void gemm_cfg(torch::Tensor a, torch::Tensor b, torch::Tensor c, int64_t m, int64_t n, int64_t k, int64_t cfg)
{
    check_operands(a, b, c, m, n, k);
    c10::OptionalDeviceGuard guard(a.device());
    const torch::Tensor ws = workspace_for(a, b, m, n, k, (int)cfg, false);
    check_status(qm_gemm_i4_ws(a.data_ptr(), b.data_ptr(), c.data_ptr(), (int)m, (int)n, (int)k, stream_of(a), (int)cfg,
                               ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? (size_t)ws.numel() : 0),
                 "quadmul.gemm_cfg");
}

// Device-side pack_b (test.py:6-15): [rows, K] int8 -> [rows, K/2] int8.
torch::Tensor pack(torch::Tensor values)
{
    TORCH_CHECK(values.is_cuda() && values.scalar_type() == torch::kInt8 && values.dim() == 2, "quadmul.pack: expects a 2-D int8 GPU tensor");
    TORCH_CHECK(values.size(1) % 2 == 0, "quadmul.pack: K must be even");
    auto v = values.contiguous();
    c10::OptionalDeviceGuard guard(v.device());
    auto out = torch::empty({v.size(0), v.size(1) / 2}, v.options());
    check_status(qm_pack_i4(v.data_ptr(), out.data_ptr(), (int)v.size(0), (int)v.size(1), stream_of(v)), "quadmul.pack");
    return out;
}

// Per-row symmetric int4 quantisation fused with the packing (no counterpart in the
// reference beyond pack_b's packing half): [rows, K] fp16 / bf16 / fp32 -> ([rows, K/2]
// int8, [rows] float32 scales = amax / 7, the row_scale of gemm_scaled).
std::tuple<torch::Tensor, torch::Tensor> quantize_pack(torch::Tensor x)
{
    TORCH_CHECK(x.is_cuda() && x.dim() == 2, "quadmul.quantize_pack: expects a 2-D GPU tensor");
    const auto t = x.scalar_type();
    TORCH_CHECK(t == torch::kFloat16 || t == torch::kBFloat16 || t == torch::kFloat32, "quadmul.quantize_pack: x must be float16, bfloat16 or float32");
    TORCH_CHECK(x.size(1) % 2 == 0, "quadmul.quantize_pack: K must be even");
    auto v = x.contiguous();
    c10::OptionalDeviceGuard guard(v.device());
    auto packed = torch::empty({v.size(0), v.size(1) / 2}, v.options().dtype(torch::kInt8));
    auto scales = torch::empty({v.size(0)}, v.options().dtype(torch::kFloat32));
    const int in = t == torch::kFloat16 ? QM_IN_F16 : (t == torch::kBFloat16 ? QM_IN_BF16 : QM_IN_F32);
    check_status(qm_quantize_pack_i4(v.data_ptr(), in, packed.data_ptr(), scales.data_ptr<float>(), (int)v.size(0), (int)v.size(1), stream_of(v)),
                 "quadmul.quantize_pack");
    return {packed, scales};
}

// The W4A4 linear layer (quadmul_amd/linear.py) in one call: quantise + pack the rows of x, then the
// GEMM with the scaled output and the bias.  What lies between the two is in one allocation.
torch::Tensor linear(torch::Tensor x, torch::Tensor weight, int64_t n, c10::optional<torch::Tensor> weight_scale, c10::optional<torch::Tensor> bias, bool bf16)
{
    const auto t = x.scalar_type();
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), "quadmul.linear: x must be a contiguous 2-D GPU tensor");
    TORCH_CHECK(t == torch::kFloat16 || t == torch::kBFloat16 || t == torch::kFloat32, "quadmul.linear: x must be float16, bfloat16 or float32");
    TORCH_CHECK(weight.is_cuda() && weight.device() == x.device() && is_byte(weight) && weight.is_contiguous(),
                "quadmul.linear: the weight must be a contiguous int8 or uint8 tensor (packed int4) on x's device");
    const int64_t m = x.size(0), k = x.size(1);
    TORCH_CHECK(n >= 0 && k % 2 == 0 && weight.numel() == n * (k / 2), "quadmul.linear: the weight must hold ", n, " rows of ", k, " / 2 bytes");
    TORCH_CHECK(m <= INT32_MAX && n <= INT32_MAX && k <= INT32_MAX, "quadmul.linear: m, n, k must fit in int32");
    check_scale(weight_scale, x, n, "weight_scale");
    const auto out = bf16 ? torch::kBFloat16 : torch::kFloat16;
    TORCH_CHECK(!bias.has_value() || (bias->device() == x.device() && bias->scalar_type() == out && bias->is_contiguous() && bias->numel() == n),
                "quadmul.linear: the bias must be a contiguous vector of ", n, " elements of the output's type on x's device");
    c10::OptionalDeviceGuard guard(x.device());
    auto y = torch::empty({m, n}, x.options().dtype(out));
    const int in = t == torch::kFloat16 ? QM_IN_F16 : (t == torch::kBFloat16 ? QM_IN_BF16 : QM_IN_F32);
    const float *const col_scale = weight_scale.has_value() ? weight_scale->data_ptr<float>() : nullptr;
    const void *const bias_ptr = bias.has_value() ? bias->data_ptr() : nullptr;
    const int y_type = bf16 ? QM_OUT_BF16 : QM_OUT_F16, align = ptr_alignment(weight, weight);
    const size_t need = qm_linear_workspace_bytes((int)m, (int)n, (int)k, in, align);
    torch::Tensor scratch;
    if (need > 0) scratch = bytes_if_there_are(need, x.options());
    if (need == 0 || scratch.defined()) {
        check_status(qm_linear_i4(x.data_ptr(), in, weight.data_ptr(), y.data_ptr(), (int)m, (int)n, (int)k, col_scale, bias_ptr, y_type, stream_of(x),
                                  need > 0 ? scratch.data_ptr() : nullptr, need),
                     "quadmul.linear");
        return y;
    }
    // The two calls it stands for, which can do with less: the packed rows, their scales and what the GEMM must have.
    const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t packed_bytes = up((size_t)m * (k / 2)), scale_bytes = up((size_t)m * sizeof(float));
    const size_t ws_bytes = qm_gemm_workspace_bytes((int)m, (int)n, (int)k, std::min(align, 256), QM_CFG_AUTO, 1);
    scratch = torch::empty({(int64_t)(packed_bytes + scale_bytes + ws_bytes)}, x.options().dtype(torch::kUInt8));
    uint8_t *const xq = scratch.data_ptr<uint8_t>();
    float *const xs = reinterpret_cast<float *>(xq + packed_bytes);
    check_status(qm_quantize_pack_i4(x.data_ptr(), in, xq, xs, (int)m, (int)k, stream_of(x)), "quadmul.linear");
    check_status(qm_gemm_i4_scaled_bias_ws(xq, weight.data_ptr(), y.data_ptr(), (int)m, (int)n, (int)k, xs, col_scale, bias_ptr, y_type, stream_of(x),
                                           QM_CFG_AUTO, ws_bytes ? xq + packed_bytes + scale_bytes : nullptr, ws_bytes),
                 "quadmul.linear");
    return y;
}

// Device-side unpack_int4_matrix (kernel.cu:389-408): [rows, K/2] bytes -> [rows, K] int8.
torch::Tensor unpack(torch::Tensor packed)
{
    TORCH_CHECK(packed.is_cuda() && is_byte(packed) && packed.dim() == 2, "quadmul.unpack: expects a 2-D int8/uint8 GPU tensor");
    auto p = packed.contiguous();
    c10::OptionalDeviceGuard guard(p.device());
    auto out = torch::empty({p.size(0), p.size(1) * 2}, p.options().dtype(torch::kInt8));
    check_status(qm_unpack_i4(p.data_ptr(), out.data_ptr(), (int)p.size(0), (int)p.size(1) * 2, stream_of(p)), "quadmul.unpack");
    return out;
}

// 16-bit activations times packed int4 weights with a scale per group of K (include/qm_abi.h: qm_gemm_grouped_i4): a new [m, n]
// tensor of x's type. x may have any distance between its rows.
int float16_type(const torch::Tensor &t, const char *what)
{
    TORCH_CHECK(t.scalar_type() == torch::kFloat16 || t.scalar_type() == torch::kBFloat16, what, " must be float16 or bfloat16");
    return t.scalar_type() == torch::kFloat16 ? QM_IN_F16 : QM_IN_BF16;
}

void check_grouped(const torch::Tensor &x, const torch::Tensor &weight, const torch::Tensor &weight_scale, int64_t group, const c10::optional<torch::Tensor> &bias)
{
    TORCH_CHECK(x.dim() == 2 && weight.dim() == 2 && weight_scale.dim() == 2, "quadmul.gemm_grouped: x, weight and weight_scale must be 2-D");
    const int64_t m = x.size(0), k = x.size(1), n = weight.size(0);
    TORCH_CHECK(m <= INT32_MAX && n <= INT32_MAX && k <= INT32_MAX, "quadmul.gemm_grouped: m, n, k must fit in int32");
    TORCH_CHECK(is_byte(weight) && weight.is_contiguous() && k % 2 == 0 && weight.size(1) == k / 2,
                "quadmul.gemm_grouped: the weight must be a contiguous [n, k / 2] int8 or uint8 tensor (packed int4), k = ", k, " even");
    TORCH_CHECK(group >= 32 && group <= INT32_MAX && group % 32 == 0, "quadmul.gemm_grouped: the group size must be a multiple of 32, got ", group);
    TORCH_CHECK(weight_scale.is_contiguous() && weight_scale.size(0) == n && weight_scale.size(1) == (k + group - 1) / group &&
                    (weight_scale.scalar_type() == torch::kFloat32 || weight_scale.scalar_type() == x.scalar_type()),
                "quadmul.gemm_grouped: the scales must be a contiguous [n, ceil(k / group)] tensor of float32 or of x's type");
    TORCH_CHECK(x.device() == weight.device() && x.device() == weight_scale.device(), "quadmul.gemm_grouped: all tensors must be on the same device");
    TORCH_CHECK(!bias.has_value() || (bias->device() == x.device() && bias->scalar_type() == x.scalar_type() && bias->is_contiguous() && bias->numel() == n),
                "quadmul.gemm_grouped: the bias must be a contiguous vector of ", n, " elements of x's type on x's device");
}

torch::Tensor gemm_grouped(torch::Tensor x, torch::Tensor weight, torch::Tensor weight_scale, int64_t group, c10::optional<torch::Tensor> bias)
{
    TORCH_CHECK(x.is_cuda(), "quadmul.gemm_grouped: expects GPU tensors");
    const int type = float16_type(x, "quadmul.gemm_grouped: x");
    check_grouped(x, weight, weight_scale, group, bias);
    const int64_t m = x.size(0), k = x.size(1), n = weight.size(0);
    c10::OptionalDeviceGuard guard(x.device());
    if ((k > 1 && x.stride(1) != 1) || (m > 1 && x.stride(0) < k)) x = x.contiguous();
    auto y = torch::empty({m, n}, x.options());
    const int64_t stride = m > 1 ? x.stride(0) : k;
    const size_t need = qm_gemm_grouped_workspace_bytes((int)m, (int)n, (int)k, (int)group, reinterpret_cast<uintptr_t>(weight.data_ptr()) & 15 ? 1 : 16);
    torch::Tensor scratch;
    if (need > 0) scratch = torch::empty({(int64_t)need}, x.options().dtype(torch::kUInt8));
    check_status(qm_gemm_grouped_i4(x.data_ptr(), type, stride, weight.data_ptr(), weight_scale.data_ptr(), weight_scale.scalar_type() == torch::kFloat32 ? QM_IN_F32 : type,
                                    (int)group, bias.has_value() ? bias->data_ptr() : nullptr, y.data_ptr(), (int)m, (int)n, (int)k, stream_of(x),
                                    need > 0 ? scratch.data_ptr() : nullptr, need),
                 "quadmul.gemm_grouped");
    return y;
}

// The paged cache in 8 bits: three tensors (codes of the keys and of the values, scales) and what says where a sequence's tokens
// are in them, checked and put together for the C interface.
qm_kv_cache kv_cache(const char *what, const torch::Tensor &k, const torch::Tensor &v, const torch::Tensor &scales)
{
    TORCH_CHECK(k.is_cuda() && k.device() == v.device() && k.device() == scales.device(), what, ": the cache must be GPU tensors on one device");
    TORCH_CHECK(k.dim() == 4 && v.dim() == 4 && k.scalar_type() == torch::kInt8 && v.scalar_type() == torch::kInt8 && k.is_contiguous() && v.is_contiguous(), what,
                ": the codes must be contiguous int8 tensors, [pages, kv_heads, page_size, head_dim] of the keys and [pages, kv_heads, head_dim, page_size] of the values");
    const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2), dim = k.size(3);
    TORCH_CHECK(v.size(0) == pages && v.size(1) == heads && v.size(2) == dim && v.size(3) == page, what,
                ": the codes of the values must be [pages, kv_heads, head_dim, page_size], of the same sizes as the keys'");
    TORCH_CHECK(scales.scalar_type() == torch::kFloat32 && scales.is_contiguous() && scales.dim() == 3 && scales.size(0) == pages && scales.size(1) == heads &&
                    scales.size(2) == 2, what, ": the scales must be a contiguous float32 tensor [pages, kv_heads, 2]");
    TORCH_CHECK(page == 16 || page == 32 || page == 64 || page == 128, what, ": the page size must be 16, 32, 64 or 128, got ", page);
    TORCH_CHECK(dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256, what, ": the head dimension must be 64, 96, 128, 192 or 256, got ", dim);
    TORCH_CHECK(pages <= INT32_MAX && heads >= 1 && heads <= 4096, what, ": at most 2^31 - 1 pages, and 1 to 4096 heads");
    qm_kv_cache c{};
    c.k = k.data_ptr(), c.v = v.data_ptr(), c.scales = scales.data_ptr<float>();
    c.pages = (int)pages, c.kv_heads = (int)heads, c.page_size = (int)page, c.head_dim = (int)dim;
    return c;
}

void kv_sequences(const char *what, qm_kv_cache &c, const torch::Tensor &k, const torch::Tensor &table, const torch::Tensor &lengths,
                  const c10::optional<torch::Tensor> &start, int64_t tokens)
{
    const auto ints = [&](const torch::Tensor &t, int64_t dims) { return t.device() == k.device() && t.scalar_type() == torch::kInt32 && t.dim() == dims && t.is_contiguous(); };
    TORCH_CHECK(ints(table, 2) && ints(lengths, 1) && table.size(0) == lengths.size(0), what,
                ": block_table [sequences, width] and lengths [sequences] must be contiguous int32 tensors on the cache's device");
    const int64_t sequences = lengths.size(0);
    TORCH_CHECK(!start.has_value() || (ints(*start, 1) && start->size(0) == sequences + 1), what,
                ": query_start must be a contiguous int32 tensor of sequences + 1 elements on the cache's device");
    TORCH_CHECK(sequences <= INT32_MAX && table.size(1) <= INT32_MAX && tokens <= INT32_MAX, what, ": sizes must fit in int32");
    TORCH_CHECK(tokens == 0 || (sequences > 0 && (start.has_value() || tokens % sequences == 0)), what,
                ": ", tokens, " tokens of ", sequences, " sequences need a query_start");
    c.block_table = table.data_ptr<int>(), c.lengths = lengths.data_ptr<int>(), c.query_start = start.has_value() ? start->data_ptr<int>() : nullptr;
    c.sequences = (int)sequences, c.table_width = (int)table.size(1);
}

int clamped(int64_t v) { return (int)std::min<int64_t>(std::max<int64_t>(v, 0), INT32_MAX); }

c10::optional<torch::Tensor> kv_append(torch::Tensor k, torch::Tensor v, torch::Tensor cache_k, torch::Tensor cache_v, torch::Tensor scales, torch::Tensor block_table,
                                       torch::Tensor lengths, c10::optional<torch::Tensor> query_start, c10::optional<torch::Tensor> q, c10::optional<torch::Tensor> cos,
                                       c10::optional<torch::Tensor> sin, bool interleaved, int64_t max_query)
{
    const char *const what = "quadmul.kv_append";
    qm_kv_cache c = kv_cache(what, cache_k, cache_v, scales);
    const int type = float16_type(k, "quadmul.kv_append: the keys");
    const auto row = [&](const torch::Tensor &t) { return t.device() == cache_k.device() && t.scalar_type() == k.scalar_type() && t.dim() == 3 && t.size(2) == c.head_dim && (t.stride(2) == 1 || t.numel() == 0); };
    TORCH_CHECK(row(k) && row(v) && k.sizes() == v.sizes() && k.size(1) == c.kv_heads, what, ": keys and values must be [tokens, ", c.kv_heads, ", ", c.head_dim,
                "] of one type on the cache's device, the last dimension contiguous");
    const int64_t tokens = k.size(0);
    kv_sequences(what, c, cache_k, block_table, lengths, query_start, tokens);
    TORCH_CHECK(!q.has_value() || (row(*q) && q->size(0) == tokens && q->size(1) >= 1 && q->size(1) <= INT32_MAX), what, ": the queries must be [", tokens, ", heads, ",
                c.head_dim, "] of the keys' type on the cache's device, the last dimension contiguous");
    TORCH_CHECK(cos.has_value() == sin.has_value(), what, ": cos and sin go together");
    if (cos.has_value()) {
        const auto table = [&](const torch::Tensor &t) { return t.device() == cache_k.device() && t.scalar_type() == torch::kFloat32 && t.dim() == 2 && t.is_contiguous(); };
        TORCH_CHECK(table(*cos) && table(*sin) && cos->sizes() == sin->sizes() && 2 * cos->size(1) <= c.head_dim && cos->size(0) >= 1 && cos->size(0) <= INT32_MAX, what,
                    ": cos and sin must be contiguous float32 tensors [1 position or more, at most ", c.head_dim / 2, "] on the cache's device");
    }
    c10::OptionalDeviceGuard guard(cache_k.device());
    c10::optional<torch::Tensor> out;
    qm_kv_new n{};
    if (q.has_value()) {
        out = torch::empty({tokens, q->size(1), q->size(2)}, q->options());
        n.q = q->data_ptr(), n.q_out = out->data_ptr(), n.heads = (int)q->size(1), n.q_token_stride = q->stride(0), n.q_head_stride = q->stride(1);
    }
    n.k = k.data_ptr(), n.v = v.data_ptr();
    n.k_token_stride = k.stride(0), n.k_head_stride = k.stride(1), n.v_token_stride = v.stride(0), n.v_head_stride = v.stride(1);
    if (cos.has_value()) n.cos = cos->data_ptr<float>(), n.sin = sin->data_ptr<float>(), n.rotary_pairs = (int)cos->size(1), n.positions = (int)cos->size(0);
    n.tokens = (int)tokens, n.dtype = type, n.interleaved = interleaved ? 1 : 0, n.max_query = clamped(max_query);
    check_status(qm_kv_append_i8(&c, &n, stream_of(cache_k)), what);
    return out;
}

torch::Tensor kv_attend(torch::Tensor q, torch::Tensor cache_k, torch::Tensor cache_v, torch::Tensor scales, torch::Tensor block_table, torch::Tensor lengths,
                        c10::optional<torch::Tensor> query_start, c10::optional<double> scale, bool causal, int64_t window, int64_t max_query, int64_t max_length)
{
    const char *const what = "quadmul.kv_attend";
    qm_kv_cache c = kv_cache(what, cache_k, cache_v, scales);
    const int type = float16_type(q, "quadmul.kv_attend: the queries");
    TORCH_CHECK(q.device() == cache_k.device() && q.dim() == 3 && q.size(2) == c.head_dim && (q.stride(2) == 1 || q.numel() == 0), what, ": the queries must be [tokens, heads, ", c.head_dim,
                "] on the cache's device, the last dimension contiguous");
    const int64_t tokens = q.size(0), heads = q.size(1);
    TORCH_CHECK(heads >= 1 && heads <= 65535 && heads % c.kv_heads == 0, what, ": the heads of the queries must be a multiple of the cache's ", c.kv_heads, ", got ", heads);
    TORCH_CHECK(window >= 0, what, ": the window must be 0 (none) or more tokens");
    kv_sequences(what, c, cache_k, block_table, lengths, query_start, tokens);
    c10::OptionalDeviceGuard guard(cache_k.device());
    auto out = torch::empty({tokens, heads, (int64_t)c.head_dim}, q.options());
    const int most = clamped(max_query), longest = clamped(max_length);
    const size_t need = qm_kv_attend_workspace_bytes(&c, (int)tokens, (int)heads, clamped(window), most, longest);
    torch::Tensor scratch;
    if (need > 0) scratch = torch::empty({(int64_t)need}, q.options().dtype(torch::kUInt8));
    check_status(qm_kv_attend_i8(&c, q.data_ptr(), type, q.stride(0), q.stride(1), out.data_ptr(), (int)tokens, (int)heads,
                                 scale.has_value() ? (float)*scale : (float)(1.0 / std::sqrt((double)c.head_dim)), causal ? 1 : 0, clamped(window), most, longest,
                                 stream_of(cache_k), need > 0 ? scratch.data_ptr() : nullptr, need),
                 what);
    return out;
}

std::tuple<torch::Tensor, torch::Tensor> kv_read(torch::Tensor cache_k, torch::Tensor cache_v, torch::Tensor scales, torch::Tensor pages, bool bf16)
{
    const char *const what = "quadmul.kv_read";
    const qm_kv_cache c = kv_cache(what, cache_k, cache_v, scales);
    TORCH_CHECK(pages.device() == cache_k.device() && pages.scalar_type() == torch::kInt32 && pages.dim() == 1 && pages.is_contiguous() && pages.size(0) <= INT32_MAX, what,
                ": the pages must be a contiguous int32 vector on the cache's device");
    c10::OptionalDeviceGuard guard(cache_k.device());
    const auto options = cache_k.options().dtype(bf16 ? torch::kBFloat16 : torch::kFloat16);
    auto k = torch::empty({pages.size(0), c.kv_heads, c.page_size, c.head_dim}, options), v = torch::empty_like(k);
    check_status(qm_kv_read_i8(&c, pages.data_ptr<int>(), (int)pages.size(0), bf16 ? QM_IN_BF16 : QM_IN_F16, k.data_ptr(), v.data_ptr(), stream_of(cache_k)), what);
    return {k, v};
}

// Dispatcher-visible form of the same op (schema + mutation annotation), so that callers
// under torch.compile / export can keep `torch.ops.quadmul.gemm(a, b, c, m, n, k)` in the
// graph.  The reference has only the pybind function (extension.cpp:26-29), which a tracer
// cannot see through.  c is written in place; nothing is returned.
void gemm_meta(const torch::Tensor &, const torch::Tensor &, torch::Tensor &, int64_t, int64_t, int64_t) {}
void gemm_op(const torch::Tensor &a, const torch::Tensor &b, torch::Tensor &c, int64_t m, int64_t n, int64_t k) { gemm(a, b, c, m, n, k); }
void gemm_scaled_meta(const torch::Tensor &, const torch::Tensor &, torch::Tensor &, int64_t, int64_t, int64_t,
                      const c10::optional<torch::Tensor> &, const c10::optional<torch::Tensor> &) {}
void gemm_scaled_op(const torch::Tensor &a, const torch::Tensor &b, torch::Tensor &d, int64_t m, int64_t n, int64_t k,
                    const c10::optional<torch::Tensor> &row_scale, const c10::optional<torch::Tensor> &col_scale)
{
    gemm_scaled(a, b, d, m, n, k, row_scale, col_scale);
}

// The mixture of experts (include/qm_abi.h: qm_moe_route, qm_gemm_experts_i4, qm_moe_mlp_i4).
int check_route(const torch::Tensor &logits, int64_t top_k, const c10::optional<torch::Tensor> &bias, int64_t groups, int64_t top_groups, int64_t group_best)
{
    TORCH_CHECK(logits.dim() == 2, "quadmul.moe_route: the logits must be [tokens, experts]");
    const auto type = logits.scalar_type();
    TORCH_CHECK(type == torch::kFloat32 || type == torch::kFloat16 || type == torch::kBFloat16, "quadmul.moe_route: the logits must be float32, float16 or bfloat16");
    const int64_t experts = logits.size(1);
    TORCH_CHECK(logits.size(0) <= INT32_MAX && experts >= 1 && experts <= QM_ROUTE_EXPERTS, "quadmul.moe_route: 1 to ", QM_ROUTE_EXPERTS, " experts, got ", experts);
    TORCH_CHECK(groups >= 1 && groups <= 64 && experts % groups == 0 && top_groups >= 1 && top_groups <= groups && (group_best == 1 || group_best == 2),
                "quadmul.moe_route: groups must divide the experts and be at most 64, top_groups at most as many, group_best 1 or 2");
    TORCH_CHECK(top_k >= 1 && top_k <= 64 && top_k <= experts / groups * top_groups, "quadmul.moe_route: top_k must be 1 to 64, and no more than the experts to choose from, got ", top_k);
    TORCH_CHECK(!bias.has_value() || (bias->device() == logits.device() && bias->scalar_type() == torch::kFloat32 && bias->is_contiguous() && bias->dim() == 1 && bias->numel() == experts),
                "quadmul.moe_route: the bias must be a contiguous float32 vector of ", experts, " elements on the logits' device");
    return type == torch::kFloat32 ? QM_IN_F32 : type == torch::kFloat16 ? QM_IN_F16 : QM_IN_BF16;
}
std::tuple<torch::Tensor, torch::Tensor> moe_route(torch::Tensor logits, int64_t top_k, c10::optional<torch::Tensor> bias, bool sigmoid, int64_t groups, int64_t top_groups,
                                                   int64_t group_best, bool renormalise, double scale)
{
    TORCH_CHECK(logits.is_cuda(), "quadmul.moe_route: expects GPU tensors");
    const int type = check_route(logits, top_k, bias, groups, top_groups, group_best);
    c10::OptionalDeviceGuard guard(logits.device());
    const int64_t tokens = logits.size(0), experts = logits.size(1);
    if ((experts > 1 && logits.stride(1) != 1) || (tokens > 1 && logits.stride(0) < experts)) logits = logits.contiguous();
    auto chosen = torch::empty({tokens, top_k}, logits.options().dtype(torch::kInt32)), weights = torch::empty({tokens, top_k}, logits.options().dtype(torch::kFloat32));
    check_status(qm_moe_route(logits.data_ptr(), type, tokens > 1 ? logits.stride(0) : experts, (int)tokens, (int)experts, (int)top_k, bias.has_value() ? bias->data_ptr<float>() : nullptr,
                              sigmoid ? QM_SCORES_SIGMOID : QM_SCORES_SOFTMAX, (int)groups, (int)top_groups, (int)group_best, renormalise, scale, chosen.data_ptr<int>(),
                              weights.data_ptr<float>(), stream_of(logits)),
                 "quadmul.moe_route");
    return {chosen, weights};
}

// One matrix of every expert, checked against the activations and put together for the C interface.
qm_expert_weights expert_weights(const char *what, const torch::Tensor &x, const torch::Tensor &weight, const torch::Tensor &scale, int64_t group, const c10::optional<torch::Tensor> &bias)
{
    TORCH_CHECK(weight.dim() == 3 && is_byte(weight) && weight.is_contiguous(), what, ": the weights must be contiguous [experts, n, k / 2] int8 or uint8 tensors (packed int4)");
    TORCH_CHECK(group >= 32 && group <= INT32_MAX && group % 32 == 0, what, ": the group size must be a multiple of 32, got ", group);
    const int64_t experts = weight.size(0), n = weight.size(1), k = weight.size(2) * 2;
    TORCH_CHECK(experts <= INT32_MAX && n <= INT32_MAX && k <= INT32_MAX, what, ": sizes must fit in int32");
    TORCH_CHECK(scale.dim() == 3 && scale.is_contiguous() && scale.size(0) == experts && scale.size(1) == n && scale.size(2) == (k + group - 1) / group &&
                    (scale.scalar_type() == torch::kFloat32 || scale.scalar_type() == x.scalar_type()),
                what, ": the scales must be contiguous [experts, n, ceil(k / group)] tensors of float32 or of x's type");
    TORCH_CHECK(weight.device() == x.device() && scale.device() == x.device(), what, ": all tensors must be on the same device");
    TORCH_CHECK(!bias.has_value() || (bias->device() == x.device() && bias->scalar_type() == x.scalar_type() && bias->is_contiguous() && bias->dim() == 2 && bias->size(0) == experts && bias->size(1) == n),
                what, ": the bias must be a contiguous [experts, n] tensor of x's type on x's device");
    return {weight.data_ptr(), scale.data_ptr(), bias.has_value() ? bias->data_ptr() : nullptr, scale.scalar_type() == torch::kFloat32 ? QM_IN_F32 : scale.scalar_type() == torch::kFloat16 ? QM_IN_F16 : QM_IN_BF16,
            (int)experts, (int)n, (int)k, (int)group};
}
void check_chosen(const char *what, const torch::Tensor &x, const torch::Tensor &chosen)
{
    TORCH_CHECK(chosen.device() == x.device() && chosen.scalar_type() == torch::kInt32 && chosen.dim() == 2 && chosen.is_contiguous() && chosen.size(0) == x.size(0), what,
                ": the chosen experts must be a contiguous int32 tensor [tokens, top_k] on x's device");
    TORCH_CHECK(chosen.size(0) <= INT32_MAX && chosen.size(1) <= INT32_MAX && chosen.numel() <= INT32_MAX, what, ": tokens times top_k must fit in int32");
}
void check_experts(const torch::Tensor &x, const torch::Tensor &chosen, const torch::Tensor &weight)
{
    TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "quadmul.gemm_experts: x must be [tokens, k] or [tokens, top_k, k]");
    check_chosen("quadmul.gemm_experts", x, chosen);
    TORCH_CHECK(x.dim() == 2 || x.size(1) == chosen.size(1), "quadmul.gemm_experts: x must have a row for each choice, or one for each token");
    TORCH_CHECK(x.size(-1) % 2 == 0 && weight.dim() == 3 && weight.size(2) * 2 == x.size(-1), "quadmul.gemm_experts: the weights must be [experts, n, k / 2], k even and x's last dimension");
}

// Rows that the kernels for few rows to an expert can load, sixteen aligned bytes at a time; others are copied first: a pass over x. The kernels that take rows at
// any address cost more: a token, 8 of 128 of 2048 x 2048, 21 us where a copy and the product are 8.8; 16 tokens 44.5, 37.5; results are the same wherever x lies.
torch::Tensor aligned_rows(torch::Tensor x)
{
    const int64_t k = x.size(-1);
    bool apart = (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) != 0;
    for (int64_t d = 0; d + 1 < x.dim(); ++d) apart |= x.size(d) > 1 && x.stride(d) % 8 != 0;
    if ((k > 1 && x.stride(-1) != 1) || (apart && k % 32 == 0)) return x.clone(at::MemoryFormat::Contiguous);
    return x;
}

torch::Tensor gemm_experts(torch::Tensor x, torch::Tensor chosen, torch::Tensor weight, torch::Tensor weight_scale, int64_t group, c10::optional<torch::Tensor> bias)
{
    TORCH_CHECK(x.is_cuda(), "quadmul.gemm_experts: expects GPU tensors");
    const int type = float16_type(x, "quadmul.gemm_experts: x");
    check_experts(x, chosen, weight);
    const qm_expert_weights w = expert_weights("quadmul.gemm_experts", x, weight, weight_scale, group, bias);
    c10::OptionalDeviceGuard guard(x.device());
    x = aligned_rows(x);
    const int tokens = (int)chosen.size(0), top_k = (int)chosen.size(1);
    auto y = torch::empty({tokens, top_k, w.n}, x.options());
    const size_t need = qm_gemm_experts_workspace_bytes(&w, tokens, top_k);
    torch::Tensor scratch;
    if (need > 0) scratch = torch::empty({(int64_t)need}, x.options().dtype(torch::kUInt8));
    check_status(qm_gemm_experts_i4(x.data_ptr(), type, x.stride(0), x.dim() == 3 ? x.stride(1) : 0, chosen.data_ptr<int>(), &w, y.data_ptr(), tokens, top_k, stream_of(x),
                                    need > 0 ? scratch.data_ptr() : nullptr, need),
                 "quadmul.gemm_experts");
    return y;
}

void check_mlp(const torch::Tensor &x, const torch::Tensor &chosen, const torch::Tensor &weights, const torch::Tensor &up, const torch::Tensor &down)
{
    TORCH_CHECK(x.dim() == 2, "quadmul.moe_mlp: x must be [tokens, hidden]");
    check_chosen("quadmul.moe_mlp", x, chosen);
    TORCH_CHECK(weights.device() == x.device() && weights.scalar_type() == torch::kFloat32 && weights.is_contiguous() && weights.sizes() == chosen.sizes(),
                "quadmul.moe_mlp: the weights of the chosen must be a contiguous float32 tensor [tokens, top_k] on x's device");
    TORCH_CHECK(up.dim() == 3 && down.dim() == 3 && x.size(1) % 2 == 0 && up.size(2) * 2 == x.size(1) && down.size(1) == x.size(1) && up.size(0) == down.size(0) && up.size(1) == 4 * down.size(2),
                "quadmul.moe_mlp: up must be [experts, 2 inner, hidden / 2], down [experts, hidden, inner / 2]");
}
torch::Tensor moe_mlp(torch::Tensor x, torch::Tensor chosen, torch::Tensor weights, torch::Tensor up, torch::Tensor up_scale, torch::Tensor down, torch::Tensor down_scale, int64_t group)
{
    TORCH_CHECK(x.is_cuda(), "quadmul.moe_mlp: expects GPU tensors");
    const int type = float16_type(x, "quadmul.moe_mlp: x");
    check_mlp(x, chosen, weights, up, down);
    const qm_expert_weights u = expert_weights("quadmul.moe_mlp", x, up, up_scale, group, c10::nullopt), d = expert_weights("quadmul.moe_mlp", x, down, down_scale, group, c10::nullopt);
    c10::OptionalDeviceGuard guard(x.device());
    x = aligned_rows(x);
    const int tokens = (int)chosen.size(0), top_k = (int)chosen.size(1);
    auto y = torch::empty({x.size(0), x.size(1)}, x.options());
    const size_t need = qm_moe_mlp_workspace_bytes(&u, &d, tokens, top_k);
    torch::Tensor scratch;
    if (need > 0) scratch = torch::empty({(int64_t)need}, x.options().dtype(torch::kUInt8));
    check_status(qm_moe_mlp_i4(x.data_ptr(), type, x.stride(0), chosen.data_ptr<int>(), weights.data_ptr<float>(), &u, &d, y.data_ptr(), tokens, top_k, stream_of(x),
                               need > 0 ? scratch.data_ptr() : nullptr, need),
                 "quadmul.moe_mlp");
    return y;
}

// quantize_pack returns new tensors: the Meta form only has to give their shapes and types
std::tuple<torch::Tensor, torch::Tensor> quantize_pack_meta(const torch::Tensor &x)
{
    TORCH_CHECK(x.dim() == 2 && x.size(1) % 2 == 0, "quadmul.quantize_pack: expects a 2-D tensor with even K");
    return {torch::empty({x.size(0), x.size(1) / 2}, x.options().dtype(torch::kInt8)), torch::empty({x.size(0)}, x.options().dtype(torch::kFloat32))};
}
std::tuple<torch::Tensor, torch::Tensor> quantize_pack_op(const torch::Tensor &x) { return quantize_pack(x); }

torch::Tensor gemm_grouped_op(const torch::Tensor &x, const torch::Tensor &weight, const torch::Tensor &weight_scale, int64_t group, const c10::optional<torch::Tensor> &bias)
{
    return gemm_grouped(x, weight, weight_scale, group, bias);
}
torch::Tensor gemm_grouped_meta(const torch::Tensor &x, const torch::Tensor &weight, const torch::Tensor &weight_scale, int64_t group, const c10::optional<torch::Tensor> &bias)
{
    float16_type(x, "quadmul.gemm_grouped: x");
    check_grouped(x, weight, weight_scale, group, bias);
    return torch::empty({x.size(0), weight.size(0)}, x.options());
}

// (two schemas: an operator whose result is None has no schema that every tracer takes)
void kv_append_op(const torch::Tensor &k, const torch::Tensor &v, torch::Tensor &cache_k, torch::Tensor &cache_v, torch::Tensor &scales, const torch::Tensor &block_table,
                  const torch::Tensor &lengths, const c10::optional<torch::Tensor> &query_start, const c10::optional<torch::Tensor> &cos,
                  const c10::optional<torch::Tensor> &sin, bool interleaved, int64_t max_query)
{
    kv_append(k, v, cache_k, cache_v, scales, block_table, lengths, query_start, c10::nullopt, cos, sin, interleaved, max_query);
}
void kv_append_meta(const torch::Tensor &, const torch::Tensor &, torch::Tensor &, torch::Tensor &, torch::Tensor &, const torch::Tensor &, const torch::Tensor &,
                    const c10::optional<torch::Tensor> &, const c10::optional<torch::Tensor> &, const c10::optional<torch::Tensor> &, bool, int64_t) {}
torch::Tensor kv_append_rotate_op(const torch::Tensor &q, const torch::Tensor &k, const torch::Tensor &v, torch::Tensor &cache_k, torch::Tensor &cache_v, torch::Tensor &scales,
                                  const torch::Tensor &block_table, const torch::Tensor &lengths, const c10::optional<torch::Tensor> &query_start,
                                  const c10::optional<torch::Tensor> &cos, const c10::optional<torch::Tensor> &sin, bool interleaved, int64_t max_query)
{
    return *kv_append(k, v, cache_k, cache_v, scales, block_table, lengths, query_start, q, cos, sin, interleaved, max_query);
}
torch::Tensor kv_append_rotate_meta(const torch::Tensor &q, const torch::Tensor &, const torch::Tensor &, torch::Tensor &, torch::Tensor &, torch::Tensor &, const torch::Tensor &,
                                    const torch::Tensor &, const c10::optional<torch::Tensor> &, const c10::optional<torch::Tensor> &, const c10::optional<torch::Tensor> &, bool, int64_t)
{
    return torch::empty(q.sizes(), q.options());
}
torch::Tensor kv_attend_op(const torch::Tensor &q, const torch::Tensor &cache_k, const torch::Tensor &cache_v, const torch::Tensor &scales, const torch::Tensor &block_table,
                           const torch::Tensor &lengths, const c10::optional<torch::Tensor> &query_start, c10::optional<double> scale, bool causal, int64_t window,
                           int64_t max_query, int64_t max_length)
{
    return kv_attend(q, cache_k, cache_v, scales, block_table, lengths, query_start, scale, causal, window, max_query, max_length);
}
torch::Tensor kv_attend_meta(const torch::Tensor &q, const torch::Tensor &, const torch::Tensor &, const torch::Tensor &, const torch::Tensor &, const torch::Tensor &,
                             const c10::optional<torch::Tensor> &, c10::optional<double>, bool, int64_t, int64_t, int64_t)
{
    return torch::empty(q.sizes(), q.options());
}

std::tuple<torch::Tensor, torch::Tensor> moe_route_op(const torch::Tensor &logits, int64_t top_k, const c10::optional<torch::Tensor> &bias, bool sigmoid, int64_t groups, int64_t top_groups,
                                                      int64_t group_best, bool renormalise, double scale)
{
    return moe_route(logits, top_k, bias, sigmoid, groups, top_groups, group_best, renormalise, scale);
}
std::tuple<torch::Tensor, torch::Tensor> moe_route_meta(const torch::Tensor &logits, int64_t top_k, const c10::optional<torch::Tensor> &bias, bool, int64_t groups, int64_t top_groups,
                                                        int64_t group_best, bool, double)
{
    check_route(logits, top_k, bias, groups, top_groups, group_best);
    return {torch::empty({logits.size(0), top_k}, logits.options().dtype(torch::kInt32)), torch::empty({logits.size(0), top_k}, logits.options().dtype(torch::kFloat32))};
}
torch::Tensor gemm_experts_op(const torch::Tensor &x, const torch::Tensor &chosen, const torch::Tensor &weight, const torch::Tensor &weight_scale, int64_t group,
                              const c10::optional<torch::Tensor> &bias)
{
    return gemm_experts(x, chosen, weight, weight_scale, group, bias);
}
torch::Tensor gemm_experts_meta(const torch::Tensor &x, const torch::Tensor &chosen, const torch::Tensor &weight, const torch::Tensor &weight_scale, int64_t group,
                                const c10::optional<torch::Tensor> &bias)
{
    float16_type(x, "quadmul.gemm_experts: x");
    check_experts(x, chosen, weight);
    TORCH_CHECK(weight_scale.dim() == 3 && group >= 32 && group % 32 == 0 && weight_scale.size(2) == (x.size(-1) + group - 1) / group, "quadmul.gemm_experts: the scales must be [experts, n, ceil(k / group)]");
    (void)bias;
    return torch::empty({chosen.size(0), chosen.size(1), weight.size(1)}, x.options());
}
torch::Tensor moe_mlp_op(const torch::Tensor &x, const torch::Tensor &chosen, const torch::Tensor &weights, const torch::Tensor &up, const torch::Tensor &up_scale, const torch::Tensor &down,
                         const torch::Tensor &down_scale, int64_t group)
{
    return moe_mlp(x, chosen, weights, up, up_scale, down, down_scale, group);
}
torch::Tensor moe_mlp_meta(const torch::Tensor &x, const torch::Tensor &chosen, const torch::Tensor &weights, const torch::Tensor &up, const torch::Tensor &, const torch::Tensor &down,
                           const torch::Tensor &, int64_t)
{
    float16_type(x, "quadmul.moe_mlp: x");
    check_mlp(x, chosen, weights, up, down);
    return torch::empty({x.size(0), x.size(1)}, x.options());
}

}  // namespace

TORCH_LIBRARY(quadmul, m)
{
    m.def("gemm(Tensor a, Tensor b, Tensor(c!) c, int m, int n, int k) -> ()");
    m.def("gemm_scaled(Tensor a, Tensor b, Tensor(d!) d, int m, int n, int k, Tensor? row_scale, Tensor? col_scale) -> ()");
    m.def("quantize_pack(Tensor x) -> (Tensor, Tensor)");
    m.def("gemm_grouped(Tensor x, Tensor weight, Tensor weight_scale, int group_size, Tensor? bias) -> Tensor");
    m.def("kv_append(Tensor k, Tensor v, Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor(c!) scales, Tensor block_table, Tensor lengths, Tensor? query_start, "
          "Tensor? cos, Tensor? sin, bool interleaved, int max_query) -> ()");
    m.def("kv_append_rotate(Tensor q, Tensor k, Tensor v, Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor(c!) scales, Tensor block_table, Tensor lengths, "
          "Tensor? query_start, Tensor? cos, Tensor? sin, bool interleaved, int max_query) -> Tensor");
    m.def("kv_attend(Tensor q, Tensor cache_k, Tensor cache_v, Tensor scales, Tensor block_table, Tensor lengths, Tensor? query_start, float? scale, bool causal, "
          "int window, int max_query, int max_length) -> Tensor");
    m.def("moe_route(Tensor logits, int top_k, Tensor? bias, bool sigmoid, int groups, int top_groups, int group_best, bool renormalise, float scale) -> (Tensor, Tensor)");
    m.def("gemm_experts(Tensor x, Tensor chosen, Tensor weight, Tensor weight_scale, int group_size, Tensor? bias) -> Tensor");
    m.def("moe_mlp(Tensor x, Tensor chosen, Tensor weights, Tensor up, Tensor up_scale, Tensor down, Tensor down_scale, int group_size) -> Tensor");
}
TORCH_LIBRARY_IMPL(quadmul, CUDA, m)
{
    m.impl("gemm", &gemm_op);
    m.impl("gemm_scaled", &gemm_scaled_op);
    m.impl("quantize_pack", &quantize_pack_op);
    m.impl("gemm_grouped", &gemm_grouped_op);
    m.impl("kv_append", &kv_append_op);
    m.impl("kv_append_rotate", &kv_append_rotate_op);
    m.impl("kv_attend", &kv_attend_op);
    m.impl("moe_route", &moe_route_op);
    m.impl("gemm_experts", &gemm_experts_op);
    m.impl("moe_mlp", &moe_mlp_op);
}
TORCH_LIBRARY_IMPL(quadmul, Meta, m)
{
    m.impl("gemm", &gemm_meta);
    m.impl("gemm_scaled", &gemm_scaled_meta);
    m.impl("quantize_pack", &quantize_pack_meta);
    m.impl("gemm_grouped", &gemm_grouped_meta);
    m.impl("kv_append", &kv_append_meta);
    m.impl("kv_append_rotate", &kv_append_rotate_meta);
    m.impl("kv_attend", &kv_attend_meta);
    m.impl("moe_route", &moe_route_meta);
    m.impl("gemm_experts", &gemm_experts_meta);
    m.impl("moe_mlp", &moe_mlp_meta);
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("gemm", &gemm, "Int4xInt4 Matrix Multiplication Kernel", py::arg("a"), py::arg("b"), py::arg("c"), py::arg("m"), py::arg("n"), py::arg("k"));
    m.def("gemm_scaled", &gemm_scaled, "Int4xInt4 GEMM with per-row and per-column fp32 scales, fp16 / bf16 output", py::arg("a"), py::arg("b"),
          py::arg("d"), py::arg("m"), py::arg("n"), py::arg("k"), py::arg("row_scale") = py::none(), py::arg("col_scale") = py::none());
    m.def("gemm_cfg", &gemm_cfg, "gemm with an explicit kernel configuration id (autotuning)");
    // (the launches of these may wait for room in the stream's queue: without the interpreter's lock)
    using nogil = py::call_guard<py::gil_scoped_release>;
    m.def("linear", &linear, "W4A4 linear layer: quantise + pack the rows of x, GEMM with scaled 16-bit float output, bias", py::arg("x"), py::arg("weight"),
          py::arg("out_features"), py::arg("weight_scale"), py::arg("bias"), py::arg("bf16"), nogil());
    m.def("gemm_grouped", &gemm_grouped, "16-bit activations x packed int4 weights with a scale per group of K", py::arg("x"), py::arg("weight"), py::arg("weight_scale"),
          py::arg("group_size"), py::arg("bias") = py::none(), nogil());
    m.def("kv_append", &kv_append, "New keys and values into the paged 8-bit cache, rotated on the way; returns the rotated queries", py::arg("k"), py::arg("v"),
          py::arg("cache_k"), py::arg("cache_v"), py::arg("scales"), py::arg("block_table"), py::arg("lengths"), py::arg("query_start") = py::none(), py::arg("q") = py::none(),
          py::arg("cos") = py::none(), py::arg("sin") = py::none(), py::arg("interleaved") = false, py::arg("max_query") = 0, nogil());
    m.def("kv_attend", &kv_attend, "Attention over the paged 8-bit cache", py::arg("q"), py::arg("cache_k"), py::arg("cache_v"), py::arg("scales"), py::arg("block_table"),
          py::arg("lengths"), py::arg("query_start") = py::none(), py::arg("scale") = py::none(), py::arg("causal") = true, py::arg("window") = 0, py::arg("max_query") = 0,
          py::arg("max_length") = 0, nogil());
    m.def("kv_read", &kv_read, "Pages of the 8-bit cache as 16-bit floats", py::arg("cache_k"), py::arg("cache_v"), py::arg("scales"), py::arg("pages"), py::arg("bf16"), nogil());
    m.def("moe_route", &moe_route, "A router's choice of experts and their weights", py::arg("logits"), py::arg("top_k"), py::arg("bias") = py::none(), py::arg("sigmoid") = false,
          py::arg("groups") = 1, py::arg("top_groups") = 1, py::arg("group_best") = 2, py::arg("renormalise") = false, py::arg("scale") = 1.0, nogil());
    m.def("gemm_experts", &gemm_experts, "Each token's row times the packed int4 weights of each of its experts", py::arg("x"), py::arg("chosen"), py::arg("weight"),
          py::arg("weight_scale"), py::arg("group_size"), py::arg("bias") = py::none(), nogil());
    m.def("moe_mlp", &moe_mlp, "The gated MLP of each token's experts, added up by weight", py::arg("x"), py::arg("chosen"), py::arg("weights"), py::arg("up"), py::arg("up_scale"),
          py::arg("down"), py::arg("down_scale"), py::arg("group_size"), nogil());
    m.def("pack", &pack, nogil(), "Pack a [rows, K] int8 tensor of int4 values into [rows, K/2] bytes on the GPU");
    m.def("quantize_pack", &quantize_pack, nogil(), "Per-row symmetric int4 quantisation of a [rows, K] float tensor, packed; returns (packed, scales)");
    m.def("unpack", &unpack, nogil(), "Unpack [rows, K/2] bytes into a [rows, K] int8 tensor on the GPU");
    m.def("num_configs", &qm_num_configs);
    m.def("config_name", [](int cfg) { const char *s = qm_config_name(cfg); return std::string(s ? s : ""); });
    m.def("select_config", &qm_select_config);
    m.def("version", []() { return std::string(qm_version()); });
}
