/*
 * C ABI of the MI355X (gfx950) packed-int4 GEMM library, libqm_hip.so.
 *
 *   C[M,N] (int32, row-major) = A[M,K] (s4) * B[N,K]^T (s4)
 *
 * A and B are packed two nibbles per byte along K: byte j of a row holds element
 * 2j in bits 0..3 and element 2j+1 in bits 4..7, two's complement (reference:
 * pack_b, test.py:6-15; unpack_int4_matrix, kernel.cu:389-408).  A is [M, K/2]
 * bytes, B is [N, K/2] bytes ("B is transposed", kernel.cu:78), C is fully
 * overwritten (kernel.cu:99-114,173).
 *
 * Plain pointers and sizes only; every pointer is a DEVICE pointer borrowed for
 * the duration of the enqueued work; `stream` is a hipStream_t passed as void*
 * (NULL = the default stream).  Every call is asynchronous, allocates nothing,
 * never synchronises and is therefore safe under HIP graph capture, as the
 * reference's harness requires (test.py:78-81).
 *
 * Every function returning int returns QM_OK (0) or a negative QM_ERR_* code;
 * qm_status_string() names it.  The reference has no error reporting at all
 * (extension.cpp:11-15 commented out, kernel.cu:282-288 commented out, unknown
 * shapes silently skipped at kernel.cu:340-385); returning a status is a
 * deliberate strengthening.
 */
#ifndef QM_ABI_H
#define QM_ABI_H

#include <stdint.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QM_OK                 0
#define QM_ERR_NULL          -1 /* a required pointer is NULL                               */
#define QM_ERR_SHAPE         -2 /* m, n or k negative, k odd, a size overflows int32, or a size the call does not take */
#define QM_ERR_CONFIG        -3 /* cfg id unknown, or that config cannot run this shape     */
#define QM_ERR_LAUNCH        -4 /* the HIP runtime refused the launch (see qm_last_hip_error) */
#define QM_ERR_ALIGN         -5 /* C is not 4-byte aligned (a 16-bit output: 2-byte), or a pointer less aligned
                                   than the call says                                        */
#define QM_ERR_DTYPE         -6 /* out_dtype is none of the QM_OUT_* values, or a type the call does not take */
#define QM_ERR_SCRATCH       -7 /* qm_gemm_i4_static: the call needs more scratch memory than
                                   QM_STATIC_SCRATCH_BYTES; others: a workspace that is too small */

#define QM_CFG_AUTO          -1 /* let the shape table / heuristic choose                   */
#define QM_CFG_RECODE        -2 /* 6-bit operands whether they pay or not, on tiles of 256 x 256:
                                   see qm_gemm_recode_bytes                                  */
#define QM_CFG_RECODE_NARROW -3 /* the same on tiles of 256 x 128                            */

/*
 * The hot path.  Replaces
 *   void wrapper(void *A, void *B, void *C, const int m, const int n, const int k,
 *                cudaStream_t stream)                 (kernel.cu:334, declared extension.cpp:6)
 * with the same seven arguments in the same order plus a status.  Unlike the
 * reference, every shape with m,n >= 0 and even k >= 0 is computed (m or n == 0
 * is a no-op, k == 0 zero-fills C).
 *
 * Seven arguments leave no room for a workspace.  On every shape whose best schedule needs
 * none -- 18 of the 42 shapes of the reference's table (kernel.cu:343-384), up to 64 rows, K below
 * one 128-nibble step -- this entry point runs exactly what qm_gemm_i4_ws runs.  It is slower than qm_gemm_i4_ws / qm_gemm_i4_static (measured, MI355X, both columns
 * of benchmarks/mi355x.md's second table) in three cases:
 *   - large products, which run on 6-bit floats when they are lent qm_gemm_recode_bytes (not qm_gemm_i4_static):
 *     22 of the table's shapes, 1.03 to 1.31 times as long here;
 *   - few output tiles and a long K, which those entry points split over several workgroups
 *     per tile through the workspace: here the best unsplit configuration runs instead.
 *     Two shapes of the reference's table are left that split K: 256 x 8192 x 28672, 56.0 to 59.3 us
 *     against 54.4 to 55.8, and 512 x 8192 x 28672, 94-105 us against 92-95 (1.02 to 1.11x);
 *   - K % 32 != 0, or A or B not 16-byte aligned: the kernel for operands at any address runs,
 *     several times slower on many rows than the zero-padded copies in a workspace.  Weight
 *     matrices of the reference's table all have K % 32 == 0.
 * A caller that can lend device memory should bind qm_gemm_i4_ws; one that cannot allocate,
 * qm_gemm_i4_static.
 */
int qm_gemm_i4(const void *A, const void *B, void *C, int m, int n, int k, void *stream);

/*
 * Same, with an explicit kernel configuration.  Replaces the compile-time choice
 * made by LAUNCH_KERNEL_IF_CONDITION / IGemmConfig (kernel.cu:321-332, 23-50)
 * from the constexpr table in configs.cu:19-689; used by the autotuner that
 * regenerates this library's per-shape table.  cfg = QM_CFG_AUTO behaves as
 * qm_gemm_i4.  Otherwise: configuration id in bits 0..15, tile raster group
 * height in bits 16..23 (0 = default), K split in bits 24..29 (0 or 1 = none;
 * above 1 only for the pipelined "q" configurations: C is zero-filled by a first
 * kernel and the partial sums are added into it with integer atomics, still
 * exact, still one enqueue on the caller's stream).  Bit 30, "q" configurations
 * only: launch one workgroup per (K split, tile) instead of the default persistent
 * grid whose workgroups each run several tiles back to back.
 */
int qm_gemm_i4_cfg(const void *A, const void *B, void *C, int m, int n, int k, void *stream, int cfg);

/*
 * The GEMM with a dequantising epilogue fused in:
 *   D[m][n] = round16( ((float)C[m][n] * row_scale[m]) * col_scale[n] )
 * where C is the exact int32 product above, both multiplications are IEEE single
 * precision in this order, and round16 rounds to nearest even into fp16 (QM_OUT_F16) or
 * bfloat16 (QM_OUT_BF16).  D is [M, N] 16-bit, row-major; row_scale is [M], col_scale is
 * [N], device pointers, either may be NULL for all ones.  No counterpart in the
 * reference's code: its README.md:7 names fused epilogues as what the kernel is for
 * (per-token activation scales x per-channel weight scales of an int4 linear layer);
 * C (4 bytes per element, most of the traffic of the int32 form) is never written.
 * Same calling rules as qm_gemm_i4.  The _cfg form takes a configuration as
 * qm_gemm_i4_cfg does (no K split; QM_ERR_CONFIG when that configuration has no scaled
 * output, see qm_config_has_scaled).
 */
#define QM_OUT_F16  1
#define QM_OUT_BF16 2
int qm_gemm_i4_scaled(const void *A, const void *B, void *D, int m, int n, int k, const float *row_scale,
                      const float *col_scale, int out_dtype, void *stream);
int qm_gemm_i4_scaled_cfg(const void *A, const void *B, void *D, int m, int n, int k, const float *row_scale,
                          const float *col_scale, int out_dtype, void *stream, int cfg);
int qm_config_has_scaled(int cfg); /* 1 / 0 */

/*
 * The two GEMMs with a caller-provided workspace (the counterpart of the workspace
 * argument of vendor GEMM libraries; the reference's wrapper, kernel.cu:334, has none
 * because its kernels never split K).  Shapes with few output tiles and a long K run
 * faster with K split over several workgroups per tile; with a workspace each split
 * stores its partial tile there with plain 16-byte stores and a second kernel adds the
 * splits up (scaling and rounding, for the scaled form), instead of 4-byte atomics into
 * C.  The second use (cfg = QM_CFG_AUTO only): large shapes whose K is not a multiple of
 * 32, or whose operands are not 16-byte aligned, get copies of A and B in the workspace
 * with every row padded with zeros to whole 128-nibble steps, and run on the pipelined
 * kernel, except where the kernel for operands at any address is faster.  Results are identical
 * to the forms without a workspace.
 *   workspace        device memory, 16-byte aligned, or NULL; used by the kernels of this
 *                    call only (in stream order): calls that may overlap on the GPU need
 *                    a workspace each, calls on one stream can share one
 *   workspace_bytes  its size; qm_gemm_workspace_bytes says how much this call can use.
 *                    A smaller (or no) workspace is not an error: the call then runs as
 *                    the form without one (except that an explicit cfg with a K split
 *                    and the scaled output returns QM_ERR_CONFIG).
 * cfg as for qm_gemm_i4_cfg (QM_CFG_AUTO included); with a workspace the scaled form also
 * takes K splits, on every "q" configuration.
 * qm_gemm_workspace_bytes: what the call with these arguments uses at most (0 when it
 * needs none, which includes calls that run on the kernel for operands at any address);
 * ptr_align is the smallest alignment in bytes shared by A and B; scaled = 1 for the scaled form.
 */
int qm_gemm_i4_ws(const void *A, const void *B, void *C, int m, int n, int k, void *stream, int cfg,
                  void *workspace, size_t workspace_bytes);
int qm_gemm_i4_scaled_ws(const void *A, const void *B, void *D, int m, int n, int k, const float *row_scale,
                         const float *col_scale, int out_dtype, void *stream, int cfg, void *workspace,
                         size_t workspace_bytes);
/* The scaled form with a bias: D[m][n] = round16(D[m][n] as above + bias[n]), bias [N] in D's
 * 16-bit type (2-byte aligned device pointer, or NULL for none) -- two roundings, the values a
 * separate in-place addition to D gives, without its pass over D. */
int qm_gemm_i4_scaled_bias_ws(const void *A, const void *B, void *D, int m, int n, int k, const float *row_scale,
                              const float *col_scale, const void *bias, int out_dtype, void *stream, int cfg,
                              void *workspace, size_t workspace_bytes);
size_t qm_gemm_workspace_bytes(int m, int n, int k, int ptr_align, int cfg, int scaled);
/*
 * The bytes of workspace with which a large product (cfg = QM_CFG_AUTO) runs faster still: A is re-coded
 * there as 6-bit floats, three quarters of a byte per element, for a matrix instruction that takes twice
 * as many of them as int8 values (and B is copied with zero-padded rows where the call would copy both operands).
 * The results are the same bit for bit.  0 where that does not pay, or
 * would take more than 256 MiB; the call itself never needs it: with a workspace of fewer bytes, it runs as
 * described above.  A caller that wants both lends the larger of the two sizes.
 * With cfg = QM_CFG_RECODE or QM_CFG_RECODE_NARROW the two calls above run on them wherever they can: K a multiple of 32 from 256 to
 * 65535, 256 columns and more, 16-byte aligned operands, a workspace of
 * qm_gemm_workspace_bytes(..., cfg, scaled) bytes; QM_ERR_CONFIG elsewhere, and from the calls that take none.
 */
size_t qm_gemm_recode_bytes(int m, int n, int k, int ptr_align, int scaled);
/* The tiles that a call with those bytes runs on: QM_CFG_RECODE, QM_CFG_RECODE_NARROW, or QM_CFG_AUTO where they are 0
 * (qm_select_config_ex then names the kernel; it names the one that runs without them elsewhere). */
int qm_recode_config(int m, int n, int k, int ptr_align, int scaled);

/*
 * qm_gemm_i4 for callers that cannot allocate and have no workspace to lend: code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc.  No counterpart in
 * the reference (its wrapper, kernel.cu:334, never needs scratch memory because it never
 * splits K and skips the shapes it has no table row for).  Runs exactly what
 * qm_gemm_i4_ws(..., QM_CFG_AUTO, workspace, bytes) runs when it is lent a workspace of
 * qm_gemm_workspace_bytes(m, n, k, align, QM_CFG_AUTO, 0) bytes -- same kernels, same result
 * bit for bit -- but the partial tiles of a K split and the zero-padded operand copies live
 * in an array of QM_STATIC_SCRATCH_BYTES that is part of the library's device code: every
 * GPU the library runs on holds one copy of it from the first kernel launch until the
 * process ends.  The call makes no hipMalloc / hipFree and no other allocating call.
 *   - A call that would use more than QM_STATIC_SCRATCH_BYTES returns QM_ERR_SCRATCH and
 *     enqueues nothing (use qm_gemm_i4_ws with a workspace of your own, or qm_gemm_i4).
 *   - All calls on one GPU share that GPU's array: calls on ONE stream are ordered and
 *     safe; calls that may overlap on the GPU (different streams, no dependency) race on
 *     it and must not both use this entry point.  Nothing in the array has to start from
 *     zero (every byte a kernel reads was written by an earlier kernel of the same call).
 *   - The first call on a device looks the array's address up (hipGetSymbolAddress); make
 *     one call per device before capturing this entry point into a graph.
 */
#define QM_STATIC_SCRATCH_BYTES (64u << 20)
int qm_gemm_i4_static(const void *A, const void *B, void *C, int m, int n, int k, void *stream);

/* The configuration qm_gemm_i4_ws picks for this shape when it is given a workspace
 * (the table lookup the reference does at kernel.cu:340-385, here with a heuristic
 * fallback instead of a silent no-op); without a workspace the K split may be lower.  ptr_align is the
 * smallest alignment in bytes shared by A and B (pass 16 or more when they come from a device
 * allocator).  "generic" (configuration 0) stands for operands that no other configuration takes:
 * called with QM_CFG_AUTO they run on the kernel for operands at any address, which has no id of its
 * own, or on zero-padded copies in the workspace, and where neither takes them (k < 32 or more than
 * 16 x 65535 rows without copies, k > 131071, operands of 2 GiB and more) on one thread per element.
 * Id 0 passed to qm_gemm_i4_cfg asks for one thread per element whatever the shape, many times slower. */
int qm_select_config(int m, int n, int k, int ptr_align);
/* The same for every form of the call: has_workspace = 0 gives what qm_gemm_i4 / qm_gemm_i4_cfg
 * (QM_CFG_AUTO) run, which never split K through a workspace; scaled = 1 the choice of the
 * qm_gemm_i4_scaled* forms. */
int qm_select_config_ex(int m, int n, int k, int ptr_align, int has_workspace, int scaled);

/* Introspection of the compiled-in configurations (the counterpart of the
 * KernelConfig instances, configs.cu:1-17). */
int         qm_num_configs(void);
const char *qm_config_name(int cfg);                       /* NULL when cfg is out of range */
int         qm_config_supports(int cfg, int m, int n, int k, int ptr_align); /* 1 / 0      */

/*
 * Device-side packing and unpacking, the steps on either side of the GEMM:
 *   qm_pack_i4   replaces pack_b (test.py:6-15):             [rows,K] int8 -> [rows,K/2] bytes
 *   qm_unpack_i4 replaces unpack_int4_matrix (kernel.cu:389-408): the inverse
 * Values outside [-8,7] are truncated to their low nibble when packing.
 */
int qm_pack_i4(const void *src_i8, void *dst_packed, int rows, int k, void *stream);
int qm_unpack_i4(const void *src_packed, void *dst_i8, int rows, int k, void *stream);

/*
 * Quantise and pack in one pass: the step before the GEMM when the activations of an int4
 * linear layer arrive as floats.  Per row r of x ([rows, k], row-major, fp16 / bf16 / fp32):
 *   amax = max_j |x[r][j]|,  scales[r] = amax / 7,
 *   q[j] = clamp(rint(x[r][j] * (7 / amax)), -7, 7)        (all zero when amax == 0)
 * in IEEE single precision with round-half-to-even, packed as qm_pack_i4 packs (the
 * packing half is pack_b, test.py:6-15; the reference has no quantiser: its test draws
 * int4 values directly, test.py:22-23).  scales is [rows] float32 and is what
 * qm_gemm_i4_scaled takes as row_scale.  x must be finite.  Each row is read from HBM once.
 */
#define QM_IN_F16  1
#define QM_IN_BF16 2
#define QM_IN_F32  3
int qm_quantize_pack_i4(const void *x, int in_dtype, void *dst_packed, float *scales, int rows, int k, void *stream);

/*
 * The int4 linear layer in one call: the rows of x quantised as qm_quantize_pack_i4 quantises them, the GEMM with the scaled
 * output on them -- D[m][n] as qm_gemm_i4_scaled_bias_ws gives it with their scales as row_scale -- and
 * the same values bit for bit as those two calls one after the other.  The reference has no counterpart.
 * Large products go from x to the 6-bit operands of qm_gemm_recode_bytes without the packed rows in between; one or two
 * rows, and up to sixteen of 16-bit types on few columns, are one launch, which wants no workspace (qm_linear_workspace_bytes is 0).
 *   workspace    device memory, 256-byte aligned, at least qm_linear_workspace_bytes(...) bytes (weight_align: the
 *                alignment of B in bytes), else QM_ERR_SCRATCH and nothing is enqueued; used in stream order by
 *                the kernels of this call only
 *   D            may overlap x (a square layer in place).  A call of one launch then is two, with a workspace of 4 m and m k / 2
 *                bytes, each rounded up to 256; with less, QM_ERR_SCRATCH
 */
size_t qm_linear_workspace_bytes(int m, int n, int k, int in_dtype, int weight_align);
int qm_linear_i4(const void *x, int in_dtype, const void *B, void *D, int m, int n, int k, const float *col_scale,
                 const void *bias, int out_dtype, void *stream, void *workspace, size_t workspace_bytes);

/*
 * 16-bit activations times packed int4 weights with a scale per group of K (no counterpart in the reference, whose
 * activations are int4 too):
 *   D[m][n] = round16( sum_g scale[n][g] * sum_{k in g} x[m][k] * B[n][k]  + bias[n] )
 * x is [m, k] fp16 or bf16 (dtype: QM_IN_F16, QM_IN_BF16) with rows `x_stride` elements apart, B [n, k / 2] bytes as
 * everywhere in this interface, scale [n, ceil(k / group)] row-major, float32 (scale_dtype = QM_IN_F32) or of x's type; groups
 * are runs of `group` consecutive k, a multiple of 32, the last one shorter where k is no multiple of it.  bias is [n] of x's type or NULL,
 * D [m, n] of x's type.  Sums are IEEE single precision, the weights take part as the integers they are; one rounding, at
 * the end.  k is even (k == 0: D is the bias, or zero).  D must not overlap x.
 *   workspace  16-byte aligned device memory of qm_gemm_grouped_workspace_bytes(...) bytes, used in stream order by the
 *              kernels of this call only (weight_align: the alignment of B in bytes; x, the scales and D may be at any address of
 *              their types); QM_ERR_SCRATCH with less, and nothing is enqueued
 * With bf16 activations the weights take part as 136 more than they are, and 136 times the sum of x is taken off: an |x| above 2^119, or an
 * infinity, makes its row of D infinite or NaN whatever the weights are.
 */
size_t qm_gemm_grouped_workspace_bytes(int m, int n, int k, int group, int weight_align);
int qm_gemm_grouped_i4(const void *x, int dtype, long long x_stride, const void *B, const void *scale, int scale_dtype, int group,
                       const void *bias, void *D, int m, int n, int k, void *stream, void *workspace, size_t workspace_bytes);

/*
 * A paged cache of keys and values in 8 bits, and attention over it (no counterpart in the reference).  A page holds
 * `page_size` tokens of every head, as int8 codes with one float32 scale per page, head and side: the value is
 * code * scale.  Codes of the values lie with the tokens of a channel together, which is the order the product with the
 * attention weights reads them in.
 *   k            [pages, kv_heads, page_size, head_dim]  int8, 16-byte aligned
 *   v            [pages, kv_heads, head_dim, page_size]  int8, 16-byte aligned
 *   scales       [pages, kv_heads, 2]                    float32, 8-byte aligned: of the keys, of the values
 *   block_table  [sequences, table_width] int32: the page of tokens i * page_size to (i + 1) * page_size - 1 of a sequence; an
 *                entry outside 0 .. pages - 1 is no page: what would be stored there is dropped, and attention passes over its tokens
 *   lengths      [sequences] int32: tokens of a sequence, the new ones included (below 1: none)
 *   query_start  [sequences + 1] int32: the new tokens of sequence s are rows query_start[s] to query_start[s + 1] - 1 of the
 *                packed tensors; NULL: every sequence has tokens / sequences of them.  They are the last tokens of their
 *                sequence: the last row is at position lengths[s] - 1.  Rows in front of position 0 are padding;
 *                rows that query_start gives to no sequence are left as they are in the outputs.
 * page_size is 16, 32, 64 or 128; head_dim 64, 96, 128, 192 or 256.  All pointers are device pointers; what the last three hold is
 * looked at by the kernels only, and no value of theirs makes one read or write outside the tensors.
 */
typedef struct qm_kv_cache {
    void *k, *v;
    float *scales;
    int pages, kv_heads, page_size, head_dim;
    const int *block_table, *lengths, *query_start;
    int sequences, table_width;
} qm_kv_cache;

/*
 * New keys and values into the cache, the keys rotated to their positions on the way; the queries, rotated, in the same call.
 * Rotation of a head at position p, for pair i of rotary_pairs: (a, b) -> (a c - b s, b c + a s) with c = cos[p][i], s = sin[p][i]
 * ([positions, rotary_pairs] float32); (a, b) are elements i and i + rotary_pairs, or 2i and 2i + 1 with interleaved = 1; further
 * elements stay as they are; rotary_pairs = 0: no rotation, else positions is 1 or more.  A position at or past `positions` gives NaN.
 * Storing, for each page, head and side, in single precision, every operation rounded by itself:
 *   scale' = max(scale, amax * (1 / 127)), amax over the new tokens of the page; scale (never below 0) counts as 0 in a page
 *            whose first token is new, which begins anew: all its other codes become 0
 *   code   = clamp(rint(value * (1 / scale')), -127, 127); the codes that the page held become rint(code * (scale / scale')).
 *            0 where scale' is below 2^-100.  Values that are not finite make scale' NaN, and attention to the page NaN.
 * k and v are [tokens, kv_heads, head_dim] fp16 or bf16, q [tokens, heads, head_dim] or NULL, each with strides of its own (in
 * elements) between tokens and between heads; q_out is [tokens, heads, head_dim] without gaps (rows of padding: 0) and may not overlap q.
 * No two sequences may be given the same page to write to.  max_query: the most new tokens a sequence has, for the choice of the grid only: any
 * value gives the same results (0 or less: one, if there are no more tokens than sequences, else as many as there can be).
 */
typedef struct qm_kv_new {
    const void *k, *v, *q;
    void *q_out;
    long long k_token_stride, k_head_stride, v_token_stride, v_head_stride, q_token_stride, q_head_stride;
    const float *cos, *sin;
    int tokens, heads, dtype, rotary_pairs, positions, interleaved, max_query;
} qm_kv_new;
int qm_kv_append_i8(const qm_kv_cache *cache, const qm_kv_new *fresh, void *stream);

/*
 * Attention of the new tokens over the cache:
 *   out[t][h] = sum_j softmax_j( scale * q[t][h] . key_j ) value_j
 * over the tokens j of t's sequence with j <= position of t (causal = 1; else all lengths[s]) and, with window > 0, j > position - window.
 * Heads of q share those of the cache in equal runs (heads a multiple of kv_heads).  A row that attends to nothing is 0.  Scores, softmax and
 * sums are in single precision.  A weight, times the scale of its value's page, enters the product with the values rounded to 11 bits (float16), or, below
 * 2^-20 of the row's largest such product, with an error of at most 2^-31 of that; the sum that weights are divided by is of unrounded
 * ones.  q [tokens, heads, head_dim] fp16 or bf16 with strides in elements; out [tokens, heads, head_dim] of its type.  max_query and max_length: the most new tokens, and the most tokens, that a sequence has: for the choice of the
 * grid only, any values give a right result (0 or less: as many as there can be, but a max_query of one, if there are no more tokens than sequences).
 *   workspace  16-byte aligned device memory of qm_kv_attend_workspace_bytes(...) bytes, used in stream order by the kernels of this
 *              call only; QM_ERR_SCRATCH with less, and nothing is enqueued
 */
size_t qm_kv_attend_workspace_bytes(const qm_kv_cache *cache, int tokens, int heads, int window, int max_query, int max_length);
int qm_kv_attend_i8(const qm_kv_cache *cache, const void *q, int dtype, long long q_token_stride, long long q_head_stride, void *out,
                    int tokens, int heads, float scale, int causal, int window, int max_query, int max_length, void *stream,
                    void *workspace, size_t workspace_bytes);

/* Pages back as fp16 or bf16 values: k and v [count, kv_heads, page_size, head_dim], both with the channels of a token together.
 * page_ids is [count] int32 on the device; an id that is no page gives NaN.  Only k, v, scales and the sizes of `cache` are used. */
int qm_kv_read_i8(const qm_kv_cache *cache, const int *page_ids, int count, int dtype, void *k, void *v, void *stream);

/*
 * A mixture of experts on packed int4 weights (no counterpart in the reference).
 *
 * A router's choice: for each of `tokens` rows of logits z ([tokens, experts], fp16, bf16 or fp32, rows `row_stride` elements apart) the top_k experts and
 * their weights, chosen [tokens, top_k] int32 and weights [tokens, top_k] float32, best first. In double precision:
 *   s = softmax(z) (QM_SCORES_SOFTMAX; a row of minus infinities: zeros) or 1 / (1 + exp(-z)) (QM_SCORES_SIGMOID);  c = s + bias ([experts] or NULL)
 *   groups       the experts in as many equal runs; with top_groups < groups only the top_groups groups of the largest worth are chosen from: the sum of their
 *                group_best (1 or 2) largest c
 *   chosen       the top_k largest c; of equal ones, and of equal groups, the one of the lower number. NaN counts as minus infinity, softmax scores
 *                without a bias go by the logits, which are in the same order
 *   weights      s of the chosen (without the bias), divided by their sum with renormalise = 1 (a sum of 0: by 1), times scale, rounded once
 * 1 to QM_ROUTE_EXPERTS experts, up to 64 groups, top_k up to 64 and to the experts of top_groups groups. A NaN logit, or one of plus infinity, makes the weights
 * of a softmax NaN; the chosen are always top_k different experts.
 */
#define QM_ROUTE_EXPERTS 1024
#define QM_SCORES_SOFTMAX 0
#define QM_SCORES_SIGMOID 1
int qm_moe_route(const void *logits, int dtype, long long row_stride, int tokens, int experts, int top_k, const float *bias, int scores, int groups, int top_groups,
                 int group_best, int renormalise, double scale, int *chosen, float *weights, void *stream);

/*
 * One matrix of every expert: weight [experts, n, k / 2] bytes packed as everywhere in this interface, scale [experts, n, ceil(k / group)] row-major, float32
 * (scale_dtype = QM_IN_F32) or of the activations' type, bias [experts, n] of their type or NULL; groups as for qm_gemm_grouped_i4.
 */
typedef struct qm_expert_weights {
    const void *weight, *scale, *bias;
    int scale_dtype, experts, n, k, group;
} qm_expert_weights;

/*
 * Each token's row times the matrix of each of its experts:
 *   y[t][j][n] = round16( sum_g scale[e][n][g] * sum_{k in g} x[t][j][k] * weight[e][n][k] + bias[e][n] ),  e = chosen[t][j]
 * and 0 where e is none of 0 .. experts - 1 (an expert on another GPU, a token of padding). x is fp16 or bf16, token_stride elements from token to
 * token and choice_stride from choice to choice (0: the same row for all of a token's choices); y [tokens, top_k, n] of its type, not overlapping x.
 * Sums are IEEE single precision, the products of fp16 with the weights exact; one rounding to 16 bits, at the end. The same expert may be
 * chosen twice by a token. tokens * top_k up to 2^31 - 64. A row of x with an infinity or a NaN has infinities or NaN in all its columns, other rows none of them.
 * bf16 comes to the matrix cores in one of two ways, by how many rows there are to an expert (32 and more in the mean: always the second), where k is a multiple of 32:
 *   few rows     the weights take part as 136 more than they are, and 136 times the sum of x is taken off, as in qm_gemm_grouped_i4: the sum of a part of a group (128 of k at
 *                most) is off by roundings of sums of (136 + |weight|) |x|, not of |weight| |x|, and a finite element above 2^112 may make infinities or NaN of its row
 *   many rows    each row is made float16 by a power of two that brings its largest element to 2^14: elements below 2^-28 of that largest are off by up to 2^-39 of it, also where
 *                the largest meet weights of zero; that power of two makes nothing infinite that sums in single precision hold
 *   workspace    16-byte aligned device memory of qm_gemm_experts_workspace_bytes(...) bytes, used in stream order by the kernels of this call only;
 *                QM_ERR_SCRATCH with less, and nothing is enqueued. The number of bytes goes by the sizes alone (the pointers of `weights` may be NULL still); 0 for sizes
 *                that the call refuses
 */
size_t qm_gemm_experts_workspace_bytes(const qm_expert_weights *weights, int tokens, int top_k);
int qm_gemm_experts_i4(const void *x, int dtype, long long token_stride, long long choice_stride, const int *chosen, const qm_expert_weights *weights, void *y,
                       int tokens, int top_k, void *stream, void *workspace, size_t workspace_bytes);

/*
 * The gated MLP of each token's experts, their outputs added up by weight:
 *   h[t][j][i] = round16( silu(a[i]) * a[inner + i] ),  a = x[t] * up[e]^T,  e = chosen[t][j];   y[t] = round16( sum_j weights[t][j] * h[t][j] * down[e]^T )
 * silu(a) = a / (1 + exp(-a)); up has n = 2 inner rows of k = hidden, down n = hidden rows of k = inner, neither a bias. Choices whose expert is none of
 * 0 .. experts - 1 add nothing, whatever their weight is; another choice's weight that is not finite leaves nothing finite in its token's row. Sums, the gates and the outputs of the experts are in
 * single precision (a gate below -88.7 gives 0: its exponential is infinite there); h is rounded to x's type, of which the second product's operands are, and y once, at the end. Both
 * products take bf16 as qm_gemm_experts_i4 does. `up` and `down` may have groups of different sizes and scales of different types. x [tokens, hidden] fp16 or bf16, y [tokens, hidden] of its type, not overlapping x; weights [tokens, top_k]
 * float32. Workspace as for qm_gemm_experts_i4, of qm_moe_mlp_workspace_bytes(...) bytes: for each choice of a token 2 inner bytes, as many again for many rows, and 4 hidden for each part that the second
 * product's K is cut into (1, up to 8 where there are few rows).
 */
size_t qm_moe_mlp_workspace_bytes(const qm_expert_weights *up, const qm_expert_weights *down, int tokens, int top_k);
int qm_moe_mlp_i4(const void *x, int dtype, long long token_stride, const int *chosen, const float *weights, const qm_expert_weights *up, const qm_expert_weights *down,
                  void *y, int tokens, int top_k, void *stream, void *workspace, size_t workspace_bytes);

/*
 * Optional: everything a first launch on the current device would otherwise do once -- the
 * LDS size attribute and the residency query of every kernel of the int4 products, the address of the library's
 * scratch array -- without launching anything (qm_gemm_grouped_i4, qm_gemm_experts_i4, qm_moe_mlp_i4 and qm_kv_attend_i8 set their kernels' LDS size
 * themselves, at the first launch, under capture too).  No counterpart in the reference (its
 * launch_igemm, kernel.cu:268-289, needs no set-up: 32 KB of shared memory at most).  First
 * launches do this by themselves, under HIP graph capture too; a caller that wants no
 * runtime queries inside a capture or a latency-critical first call makes this call first,
 * once per device, with that device current.
 */
int qm_init(void);

/*
 * Testing aid, not for production callers.  Operands of 2 GiB and more are cut by the library
 * into blocks its kernels' 32-bit row offsets reach: blocks of rows of A, and blocks of rows
 * of B, which are blocks of columns of C written through a row stride.  This call lowers that
 * limit (bytes; <= 0 restores 2^31 - 1) so that the block paths can be driven on small
 * shapes; it returns the previous limit.  Process-wide, not synchronised with calls in
 * flight on other threads.  No counterpart in the reference (its kernels take no operand
 * beyond their table's shapes, kernel.cu:340-385).
 */
long long qm_debug_set_operand_limit(long long bytes);

/* Diagnostics.  qm_version names the compiler the library was built with: the kernels
 * manage matrix-core hazards by hand, so a result is validated for that compiler. */
const char *qm_status_string(int status);
int         qm_last_hip_error(void);      /* hipError_t of the last failed launch on this thread */
const char *qm_version(void);

#ifdef __cplusplus
}
#endif
#endif /* QM_ABI_H */
