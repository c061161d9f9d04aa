/*
 * reef_hip: int8 attention for AMD MI355X (gfx950), C ABI.
 *
 * Drop-in device back end for the Reef engine's attention and quantization
 * operators (inference-engine/reference/cpp/include/inference_engine/). Every
 * entry point names the engine function whose arithmetic it follows, in the
 * way the engine's kernel ABI does (coral/include/reef_kernels/kernels.hpp:3-16):
 *
 *   - The caller owns every buffer; pointers are device pointers, arrays are
 *     row-major, and the innermost (head_dim / width) dimension is contiguous.
 *     Nothing here allocates or keeps hidden state, so calls are stream-ordered
 *     and re-entrant (kernels.hpp:13-14).
 *   - Where the engine throws, an entry point returns a status instead
 *     (kernels.hpp has no error path; host_if.hpp:24-30 uses status codes). All
 *     shape and argument checks run on the host before any launch.
 *   - Conditions only the device can see (non-finite values, out-of-range page
 *     numbers) set bits in an optional caller-owned device word (status_word);
 *     reef_read_status_word() waits for the stream and maps the word to a
 *     status. The C++ wrapper attention.hpp turns statuses into the engine's
 *     exception types.
 *
 * Scores follow the engine's W8A8 dequantization order
 * (operator/linear.hpp:125-127): s = float(int32 q.k) * (s_q * s_k), times
 * softmax_scale (1 reproduces the engine's unscaled attend_head,
 * attention.hpp:102-106; 1/sqrt(head_dim) is scaled dot-product attention).
 */
#ifndef REEF_HIP_ATTENTION_H
#define REEF_HIP_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum reef_status {
    REEF_OK = 0,
    /* engine: std::invalid_argument for shapes and masks
     * (activation.hpp:178-181, 204-207; attention.hpp:293-318). */
    REEF_INVALID_ARGUMENT = 1,
    /* engine: std::invalid_argument from quantize_int8 (quant.hpp:72-74). */
    REEF_NON_FINITE_INPUT = 2,
    /* engine: std::length_error for the KV cache (attention.hpp:321-327). */
    REEF_CAPACITY = 3,
    /* a HIP runtime call failed. */
    REEF_HIP_ERROR = 4,
    /* well-formed but outside what the kernels implement (e.g. head_dim). */
    REEF_UNSUPPORTED = 5,
    /* engine: std::overflow_error from safe_multiply / safe_add (util.hpp:81-131). */
    REEF_OVERFLOW = 6
} reef_status;

/* Bits set in a status word by the kernels. */
#define REEF_STATUS_BIT_NON_FINITE 0x1u
#define REEF_STATUS_BIT_BAD_PAGE 0x2u
#define REEF_STATUS_BIT_BAD_LENGTH 0x4u
#define REEF_STATUS_BIT_CAPACITY 0x8u
#define REEF_STATUS_BIT_OVERFLOW 0x10u

typedef enum reef_scale_granularity {
    REEF_SCALE_PER_TENSOR = 0, /* one scale: scales[0] */
    REEF_SCALE_PER_HEAD = 1,   /* scales[head], over batch and tokens */
    REEF_SCALE_PER_TOKEN = 2   /* scales[(b * heads + head) * tokens + t] */
} reef_scale_granularity;

/* Element strides of a [batch, heads, tokens, head_dim] tensor whose head_dim
 * is contiguous. NULL means the packed layout {H*S*D, S*D, D}. The engine keeps
 * heads as [1, heads, len, head_dim] (attention.hpp:49-68); a projection
 * output [len, heads * head_dim] is {0, D, H*D}. */
typedef struct reef_strides {
    int64_t batch, head, token;
} reef_strides;

/* ---------------------------------------------------------------------------
 * Quantization (quant.hpp): scale = max|x| / 127 (1 when max is 0), code =
 * clamp(nearbyint(x / scale), -127, 127), IEEE division, ties to even. The
 * codes and scales are bit-identical to the engine's.
 */

/* The quant.hpp rule with one scale over all n values. scale: 1 float. */
reef_status reef_quantize_int8_per_tensor(const float *x, int64_t n, int8_t *q, float *scale,
                                          uint32_t *status_word, hipStream_t stream);

/* x: [B, H, S, D] with x_strides (NULL = packed); q: packed [B, H, S, D];
 * scales: [H], each over x[:, h, :, :]. */
reef_status reef_quantize_int8_per_head(const float *x, int64_t batch, int64_t heads,
                                        int64_t tokens, int64_t head_dim,
                                        const reef_strides *x_strides, int8_t *q, float *scales,
                                        uint32_t *status_word, hipStream_t stream);

/* quantize_rows (quant.hpp:112-133), the per-token quantizer of the W8A8
 * linear (linear.hpp:120): rows of width values, row r at x + r * row_stride;
 * q packed [rows, width]; scales [rows]. */
reef_status reef_quantize_int8_per_token(const float *x, int64_t rows, int64_t width,
                                         int64_t row_stride, int8_t *q, float *scales,
                                         uint32_t *status_word, hipStream_t stream);

/* The same rows out of a strided [B, H, S, D] tensor (NULL: packed), in [B, H, S]
 * order: q packed [B, H, S, D], scales [B, H, S]. Whole 16-byte rows only (head_dim and
 * strides multiples of 4, x on 16 bytes, head_dim at most 1024) and fewer than 2^31 of
 * them: REEF_UNSUPPORTED otherwise. */
reef_status reef_quantize_int8_per_token_heads(const float *x, int64_t batch, int64_t heads,
                                               int64_t tokens, int64_t head_dim,
                                               const reef_strides *x_strides, int8_t *q,
                                               float *scales, uint32_t *status_word,
                                               hipStream_t stream);

/* Dequantize: x[i] = float(q[i]) * scale[i / group] (group = width for
 * per-token rows, n for per-tensor). */
reef_status reef_dequantize_int8(const int8_t *q, int64_t n, int64_t group, const float *scales,
                                 float *x, hipStream_t stream);

/* Waits for the stream, reads a status word written by the kernels and maps
 * it: 0 -> REEF_OK, NON_FINITE -> REEF_NON_FINITE_INPUT, CAPACITY ->
 * REEF_CAPACITY, OVERFLOW -> REEF_OVERFLOW, page/length bits ->
 * REEF_INVALID_ARGUMENT (first match in that order). Clears the word afterwards
 * when clear != 0. */
reef_status reef_read_status_word(uint32_t *status_word, int clear, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * W8A8 projection: linear() with a QuantizedWeight (operator/linear.hpp:106-132).
 * x [rows, in] fp32 (row r at x + r * x_row_stride) is quantized per row as
 * quantize_rows does (quant.hpp:112-133), multiplied by the int8 weight
 * [out, in] (row-major, the engine's layout) in exact int32, and
 * y[r, c] = float(sum) * (row_scale[r] * w_scales[c]) (+ bias[c]), the engine's
 * float steps in its order, each rounded on its own: bit-identical outputs. y is
 * fp32 [rows, out] with row stride y_row_stride. in must be a multiple of 16.
 * Non-finite input sets NON_FINITE; an infinite or NaN output sets OVERFLOW
 * (the engine's std::overflow_error). The workspace holds the quantized rows.
 */
size_t reef_linear_w8a8_workspace_bytes(int64_t rows, int64_t in_features);

reef_status reef_linear_w8a8(const float *x, int64_t rows, int64_t in_features,
                             int64_t x_row_stride, const int8_t *weight, const float *w_scales,
                             const float *bias, int64_t out_features, float *y,
                             int64_t y_row_stride, void *workspace, size_t workspace_bytes,
                             uint32_t *status_word, hipStream_t stream);

/* The product and epilogue alone, on rows already quantized (xq [rows, in] packed,
 * x_scales [rows]). */
reef_status reef_gemm_w8a8(const int8_t *xq, const float *x_scales, int64_t rows,
                           int64_t in_features, const int8_t *weight, const float *w_scales,
                           const float *bias, int64_t out_features, float *y,
                           int64_t y_row_stride, uint32_t *status_word, hipStream_t stream);

/* The same two with an epilogue, y = activation(float(sum) * (row_scale * w_scale) + bias)
 * + residual, every float step rounded on its own (with REEF_ACT_NONE and no residual, the
 * outputs of the calls above bit for bit). GELU_TANH is the engine's form
 * x / (1 + exp(-2 sqrt(2 / pi) (x + 0.044715 x^3))), GELU_ERF x erfc(-x / sqrt(2)) / 2, SILU
 * x / (1 + exp(-x)). residual: fp32 [rows, out], row r at residual + r *
 * residual_row_stride; it may be y itself (same pointer and stride), not overlap it
 * otherwise. An infinite or NaN value before the activation or after the residual sets
 * OVERFLOW. epilogue NULL: none. */
typedef enum reef_activation {
    REEF_ACT_NONE = 0,
    REEF_ACT_RELU = 1,
    REEF_ACT_GELU_TANH = 2,
    REEF_ACT_GELU_ERF = 3,
    REEF_ACT_SILU = 4
} reef_activation;

typedef struct reef_epilogue {
    const float *residual; /* NULL: none */
    int64_t residual_row_stride;
    int64_t activation; /* reef_activation */
} reef_epilogue;

reef_status reef_linear_w8a8_epilogue(const float *x, int64_t rows, int64_t in_features,
                                      int64_t x_row_stride, const int8_t *weight,
                                      const float *w_scales, const float *bias,
                                      const reef_epilogue *epilogue, int64_t out_features,
                                      float *y, int64_t y_row_stride, void *workspace,
                                      size_t workspace_bytes, uint32_t *status_word,
                                      hipStream_t stream);

reef_status reef_gemm_w8a8_epilogue(const int8_t *xq, const float *x_scales, int64_t rows,
                                    int64_t in_features, const int8_t *weight,
                                    const float *w_scales, const float *bias,
                                    const reef_epilogue *epilogue, int64_t out_features, float *y,
                                    int64_t y_row_stride, uint32_t *status_word,
                                    hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Root-mean-square norm of a residual sum, as the int8 rows that reef_gemm_w8a8 reads:
 * h = x + residual (fp32, one rounding; residual NULL: h = x), y = h * weight /
 * sqrt(mean(h^2) + eps) over each row of `width` values (weight NULL: ones), scale =
 * float(max|y| / 127) (1 where that is 0), code = rint(y / scale), ties to even, y unrounded
 * (64-bit steps). q: packed [rows, width]; scales: [rows]. sum (NULL allowed, with a
 * residual only) receives h; it may be x or residual itself (same pointer and stride), not
 * overlap them otherwise. Any width and any stride of at least width; eps >= 0. A
 * non-finite value of a row sets NON_FINITE, a scale beyond fp32 OVERFLOW; that row's codes
 * are unspecified.
 */
reef_status reef_rmsnorm_quantize_int8(const float *x, int64_t rows, int64_t width,
                                       int64_t x_row_stride, const float *residual,
                                       int64_t residual_row_stride, const float *weight,
                                       double eps, int8_t *q, float *scales, float *sum,
                                       int64_t sum_row_stride, uint32_t *status_word,
                                       hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Attention over int8 Q/K/V with an fp32 softmax and fp32 output.
 */

/* Attention flags. */
#define REEF_ATTN_PRECISE_PV 0x1u /* P.V with P split into fp16 hi + lo parts (22
                                     * bits) whatever the values. Without it the packed
                                     * schedule splits wherever a head's dequantized
                                     * values reach above 1 in magnitude, the other
                                     * schedules always; at or below 1 one fp16 P moves
                                     * an output by at most 2^-11 max|v_j - out| <=
                                     * 9.8e-4. Either
                                     * way each P carries an exponent offset that keeps
                                     * it out of the fp16 subnormals, so small weights
                                     * keep their precision */
/* Prefill work schedule (bits 4-6 of flags). AUTO lets the library choose from the
 * grid size and the workspace; the others force one schedule, for callers that
 * tune it and for tests that must reach every path. A forced schedule that the
 * call cannot use (BALANCED without a large enough workspace, SPLIT with PER_TOKEN
 * K/V scales, PACKED without head_dim 128, per-tensor or per-head K/V scales and a
 * workspace) returns REEF_INVALID_ARGUMENT, and PACKED outside the packed kernel's
 * limits REEF_UNSUPPORTED. AUTO takes PACKED for head_dim 128 with at least one
 * pair of 256-row query tiles per compute unit (and a workspace that holds the
 * image); of the others BALANCED, with a large enough workspace, for at most one
 * 128-row query tile per compute unit whose heaviest has many more keys than an equal
 * share, or whose tiles are equal and fill every unit (with PER_TOKEN K/V scales for
 * every such grid); otherwise SPLIT for head_dim
 * 128 and for such small grids, ONE_ITEM for head_dim 64 and with PER_TOKEN K/V
 * scales. Every schedule splits P into hi + lo where the values need it. */
#define REEF_ATTN_SCHED_MASK 0x70u
#define REEF_ATTN_SCHED_AUTO 0x00u
#define REEF_ATTN_SCHED_ONE_ITEM 0x10u /* one 128-row query tile per workgroup */
#define REEF_ATTN_SCHED_SPLIT 0x20u    /* persistent workgroups; two 4-wave groups split
                                        * each tile's keys; hi + lo P */
#define REEF_ATTN_SCHED_BALANCED 0x30u /* equal (tile, key block) ranges per workgroup,
                                        * two 4-wave groups splitting each range's key
                                        * tiles (one with PER_TOKEN K/V scales); cut
                                        * tiles merge through the workspace; hi + lo P */
#define REEF_ATTN_SCHED_PACKED 0x40u   /* head_dim 128, per-tensor / per-head K and V
                                        * scales: V packed once into an fp16 image in the
                                        * workspace, 128-row query tiles, persistent
                                        * workgroups taking (light, heavy) tile pairs
                                        * from per-XCD queues in the workspace */

typedef struct reef_attention_params {
    int64_t batch, q_heads, kv_heads; /* q head h reads kv head h / (q_heads / kv_heads) */
    int64_t q_len, kv_len, head_dim;  /* head_dim 64 or 128 */
    int64_t query_start; /* position of query row 0; engine: kv_len - q_len (attention.hpp:415) */
    int64_t window;      /* 0: GlobalAttention; > 0: LocalAttention window (attention.hpp:223-261) */
    float softmax_scale;    /* > 0; scales must be positive, as the quantizers make them */
    int32_t q_granularity;  /* reef_scale_granularity of q_scales */
    int32_t kv_granularity; /* reef_scale_granularity of k_scales and v_scales */
    uint32_t flags;
} reef_attention_params;

/* Prefill / general attention: Attention::context (attention.hpp:374-432) for
 * every (batch, head) in one launch; per head, attend_head (:117-123) with
 * causal_visibility (:82-100). q [B, Hq, q_len, D], k and v [B, Hkv, kv_len, D],
 * out fp32 [B, Hq, q_len, D], each with optional strides. Requires
 * query_start + q_len <= kv_len, so that every row sees a key (the engine
 * throws for a row with none, activation.hpp:204-207).
 *
 * workspace (optional, 256-byte aligned, at least
 * reef_attention_prefill_workspace_bytes(p) bytes; NULL/0 allowed) holds the
 * counters (a fixed 256 KB region: the balanced schedule's, at most 65520 items of
 * 128 query rows, and the packed schedule's item queue) and partial results of the
 * balanced schedule and, for head_dim 128, the fp16 value image of the packed
 * schedule (2 bytes per V element). It must be zero-filled
 * before its first use; every call leaves the counters zero-filled, and the
 * counters sit at the same offsets for every shape, so one workspace serves calls
 * of any shape that it is large enough for. Without it the library uses the
 * schedules that need none. Calls that may run at the same time need separate
 * workspaces. */
size_t reef_attention_prefill_workspace_bytes(const reef_attention_params *p);

reef_status reef_attention_prefill_int8(const reef_attention_params *p, const int8_t *q,
                                        const reef_strides *q_strides, const int8_t *k,
                                        const reef_strides *k_strides, const int8_t *v,
                                        const reef_strides *v_strides, const float *q_scales,
                                        const float *k_scales, const float *v_scales, float *out,
                                        const reef_strides *out_strides, void *workspace,
                                        size_t workspace_bytes, hipStream_t stream);

/* Bit-exact hook: the int32 score accumulators q . k^T (tensor.hpp:210-246
 * with int8 inputs and int32 sums), computed by the same MFMA tile code as the
 * prefill kernel. acc: [B, Hq, q_len, kv_len] int32. Packed q and k. */
reef_status reef_qk_scores_i32(const int8_t *q, const int8_t *k, int64_t batch, int64_t q_heads,
                               int64_t kv_heads, int64_t q_len, int64_t kv_len, int64_t head_dim,
                               int32_t *acc, hipStream_t stream);

/* The same scores from the packed schedule's own kernel (head_dim 128; the
 * matmul<int8_t, int32_t> of tensor.hpp:210-246 on q . k^T): it runs one attention
 * over (q, k, v = k) in which every row sees every key, and stores every score
 * accumulator as its tile code reads it (keys staged in LDS in its permuted order,
 * accumulators relative to the running maximum), turned back into the plain int32
 * sum. acc: [B, Hq, q_len, kv_len] int32; packed q [B, Hq, q_len, 128] and k
 * [B, Hkv, kv_len, 128]; workspace: 256-byte aligned, zero-filled once (the launch
 * leaves it zero-filled where it must be), at least
 * reef_qk_scores_i32_packed_workspace_bytes() bytes (0: invalid sizes). A test hook. */
size_t reef_qk_scores_i32_packed_workspace_bytes(int64_t batch, int64_t q_heads,
                                                 int64_t kv_heads, int64_t q_len,
                                                 int64_t kv_len);
reef_status reef_qk_scores_i32_packed(const int8_t *q, const int8_t *k, int64_t batch,
                                      int64_t q_heads, int64_t kv_heads, int64_t q_len,
                                      int64_t kv_len, int32_t *acc, void *workspace,
                                      size_t workspace_bytes, hipStream_t stream);

/* Integer-only attention: attend_head_int8 (int8.hpp:250-279) for every (batch,
 * head) in one launch, bit-identical to the engine. Per row: int32 scores over the
 * visible keys, weights table[min((max - s) >> score_shift, 255)], probabilities
 * in [0, 255] from the integer reciprocal of their sum (masked_softmax_int8,
 * :180-232), out = saturate_int8(rounding_shift(sum p * v, out_shift)) (:43-60).
 * table: 256 uint16 on the device (exp_table(), :156-164). q, k, v int8
 * [B, H, S, D] with strides as for the prefill; out int8 [B, Hq, q_len, D].
 * p->softmax_scale, q_granularity, kv_granularity and flags are not used;
 * head_dim 32, 64 or 128; score_shift and out_shift at most 31. A row may see at
 * most 65536 keys (kv_len, or the window when shorter): beyond that the engine's
 * uint32 weight sum could wrap, and the call returns REEF_UNSUPPORTED. */
reef_status reef_attention_int8_integer(const reef_attention_params *p, const int8_t *q,
                                        const reef_strides *q_strides, const int8_t *k,
                                        const reef_strides *k_strides, const int8_t *v,
                                        const reef_strides *v_strides, uint32_t score_shift,
                                        const uint16_t *table, uint32_t out_shift, int8_t *out,
                                        const reef_strides *out_strides, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Decode over an int8 KV cache (one query token per sequence), split across
 * waves along the keys, partial results combined by log-sum-exp.
 *
 * KV cache format (int8 values, fp32 per-token-per-head scales). The cache is
 * cut into pages of 16 tokens. A K page is [16, D] (token-major, like the
 * engine's KvCache rows, attention.hpp:64-68). A V page is stored transposed,
 * [D, 16]: each of its D rows holds one channel of the 16 tokens, which is the
 * operand layout of the P.V matrix instruction. reef_kv_pack_v_pages() converts
 * token-major values into this layout and reef_kv_append_int8() writes it.
 *
 *   contiguous: k_cache [B, Hkv, L, D]; v_cache [B, Hkv, L/16, D, 16];
 *               k_scales, v_scales [B, Hkv, L]; L = max_context, a multiple of 16.
 *   paged:      k_pages [P, Hkv, 16, D]; v_pages [P, Hkv, D, 16];
 *               k_scale_pages, v_scale_pages [P, Hkv, 16];
 *               block_table [B, max_blocks_per_seq] int32 page numbers.
 * q: [B, Hq, D] int8 with q_scales by q_granularity (PER_TOKEN: [B, Hq]);
 * out: [B, Hq, D] fp32. context_lens: [B] int32 on the device (NULL: every
 * sequence holds max_context tokens). Query b sits at position
 * context_lens[b] - 1 and sees all earlier keys (or the last window).
 * A sequence whose length is outside [1, max_context], or a page number outside
 * [0, P), sets a status-word bit and yields zeros for that sequence.
 */
typedef struct reef_decode_params {
    int64_t batch, q_heads, kv_heads, head_dim; /* head_dim 64 or 128 */
    int64_t max_context;  /* tokens per sequence the cache can hold */
    int64_t window;       /* 0: global */
    float softmax_scale;
    int32_t q_granularity;
    int32_t num_splits;   /* 0: library choice; n > 0: about n waves per (sequence,
                             kv head) on average (ceil(B * Hkv * n / 4) workgroups) */
    uint32_t flags;
} reef_decode_params;

/* Bytes of device workspace the decode entry points need for params. The launch
 * deals the keys of all (sequence, kv head) items out to its workgroups in equal
 * runs of 64-key blocks, whatever the context lengths (with at most 2048 items;
 * beyond that, in equal runs of whole items). The workspace holds a fixed 8 KB
 * region of counters (one per item, at the same offset for every shape) and two
 * partial-result slots per workgroup; an item whose keys span several workgroups
 * is merged by the last of them inside the same launch. The workspace must be
 * zero-filled before its first use; every call leaves it ready for the next call of
 * any shape it is large enough for (no refill). Calls that may run at the same
 * time need separate workspaces. */
size_t reef_attention_decode_workspace_bytes(const reef_decode_params *p);

reef_status reef_attention_decode_int8(const reef_decode_params *p, const int8_t *q,
                                       const float *q_scales, const int8_t *k_cache,
                                       const int8_t *v_cache, const float *k_scales,
                                       const float *v_scales, const int32_t *context_lens,
                                       float *out, void *workspace, size_t workspace_bytes,
                                       uint32_t *status_word, hipStream_t stream);

reef_status reef_attention_decode_int8_paged(
    const reef_decode_params *p, const int8_t *q, const float *q_scales, const int8_t *k_pages,
    const int8_t *v_pages, const float *k_scale_pages, const float *v_scale_pages,
    const int32_t *block_table, int64_t max_blocks_per_seq, int64_t num_pages,
    const int32_t *context_lens, float *out, void *workspace, size_t workspace_bytes,
    uint32_t *status_word, hipStream_t stream);

/* Allocation-free form of reef_attention_decode_int8_paged, with no counterpart in
 * the reference: for callers that cannot allocate or pass device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc). The
 * split-merge workspace is a fixed 16 MiB array inside the library, one per GPU,
 * held until the process ends; a call whose workspace
 * (reef_attention_decode_workspace_bytes) would exceed it returns REEF_UNSUPPORTED
 * before any launch. Each call clears the counters it uses with a small fill
 * kernel on `stream`, then runs the same kernels as the workspace entry point
 * (bit-identical outputs). Every call on one GPU shares that array: calls that
 * overlap on one GPU (other streams, other host threads) race and must not run
 * concurrently. Nothing is allocated or freed. */
reef_status reef_attention_decode_int8_paged_noalloc(
    const reef_decode_params *p, const int8_t *q, const float *q_scales, const int8_t *k_pages,
    const int8_t *v_pages, const float *k_scale_pages, const float *v_scale_pages,
    const int32_t *block_table, int64_t max_blocks_per_seq, int64_t num_pages,
    const int32_t *context_lens, float *out, uint32_t *status_word, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Attention of a tree of drafted tokens over the int8 cache (speculative decoding; also a
 * chain of a few new tokens per sequence, of lengths that differ): the T = draft_len tokens
 * of every sequence, whose keys and values the cache already holds in its last T places
 * (reef_kv_append_int8), each see the tokens before them and their own ancestors.
 *
 * q: [B, Hq, T, D] int8 with optional strides (multiples of 16; a projection [B, T, Hq * D]
 * is {T*Hq*D, D, Hq*D}), q_scales by q_granularity (PER_TOKEN: [B, Hq, T]); out: [B, Hq, T,
 * D] fp32 with optional strides (multiples of 4, 16-byte aligned). The cache, block table
 * and scales as for decode. context_lens: [B] int32 on the device, the drafted tokens
 * counted in (NULL, contiguous cache only: max_context). tree_mask: [B, T] uint64 on the
 * device; bit j of tree_mask[b][i] is set where row i sees drafted token j, itself among
 * them (bits from T on are ignored); NULL: a chain, row i sees drafted tokens 0 .. i. A row
 * whose mask is 0 is padding: zeros. With a window, row i sits at position P + (set bits of
 * its mask) - 1, P = context_lens[b] - T, as do the drafted tokens, and sees the last
 * `window` positions up to its own. Pages that hold only tokens before every row's window
 * are not looked up.
 * A sequence whose length is outside [T, max_context] sets BAD_LENGTH and yields zeros; a
 * page number outside [0, P) sets BAD_PAGE and its tokens take no part. A drafted token
 * whose scales are not finite leaves the rows that see it not finite, and no others. Scales
 * are positive, as the quantizers make them; with a query scale of 0 all that the row sees
 * has the same weight. A row's error is relative to the largest value scale among the tokens
 * that it sees itself: finite ones of any size elsewhere do not change it.
 *
 * Workspace as for decode: reef_attention_decode_tree_workspace_bytes(p) bytes (0: invalid
 * or unsupported sizes), 16-byte aligned, zero-filled before its first use; every call
 * leaves it ready for the next of any shape it is large enough for. Calls that may run at
 * the same time need separate workspaces.
 */
typedef struct reef_tree_params {
    int64_t batch, q_heads, kv_heads, head_dim; /* head_dim 64 or 128 */
    int64_t draft_len;   /* tokens per sequence, 1 .. 64 */
    int64_t max_context; /* tokens per sequence the cache can hold, a multiple of 16 */
    int64_t window;      /* 0: global */
    float softmax_scale; /* > 0 */
    int32_t q_granularity;
    uint32_t flags; /* 0 */
    uint32_t reserved;
} reef_tree_params;

size_t reef_attention_decode_tree_workspace_bytes(const reef_tree_params *p);

reef_status reef_attention_decode_tree_int8(
    const reef_tree_params *p, const int8_t *q, const reef_strides *q_strides,
    const float *q_scales, const int8_t *k_cache, const int8_t *v_cache, const float *k_scales,
    const float *v_scales, const int32_t *context_lens, const uint64_t *tree_mask, float *out,
    const reef_strides *out_strides, void *workspace, size_t workspace_bytes,
    uint32_t *status_word, hipStream_t stream);

reef_status reef_attention_decode_tree_int8_paged(
    const reef_tree_params *p, const int8_t *q, const reef_strides *q_strides,
    const float *q_scales, const int8_t *k_pages, const int8_t *v_pages,
    const float *k_scale_pages, const float *v_scale_pages, const int32_t *block_table,
    int64_t max_blocks_per_seq, int64_t num_pages, const int32_t *context_lens,
    const uint64_t *tree_mask, float *out, const reef_strides *out_strides, void *workspace,
    size_t workspace_bytes, uint32_t *status_word, hipStream_t stream);

/* Token-major values [pages * 16, D] (page-contiguous) -> transposed pages
 * [pages, D, 16]. */
reef_status reef_kv_pack_v_pages(const int8_t *v_tokens, int64_t pages, int64_t head_dim,
                                 int8_t *v_pages, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * KV-cache append: Attention::append_kv_cache (attention.hpp:290-352) on the
 * int8 cache above. The new_tokens fresh key and value rows of every sequence,
 * fp32 [B, Hkv, new_tokens, D] with optional strides (a projection output
 * [new_tokens, Hkv * D] is {0, D, Hkv * D}), are quantized per token exactly as
 * quantize_rows (quant.hpp:112-133) quantizes them and written at positions
 * start_positions[b] .. start_positions[b] + new_tokens - 1 of sequence b, in
 * place. start_positions: [B] int32 on the device.
 *   - REEF_CAPACITY (host) when new_tokens > max_context; a sequence whose
 *     append would pass max_context is not written and sets the CAPACITY bit
 *     (the engine's length_error, attention.hpp:321-327); a negative start sets
 *     BAD_LENGTH; a page number outside [0, num_pages) sets BAD_PAGE and skips
 *     that row.
 *   - Non-finite values set NON_FINITE (the engine throws before writing; here
 *     the rows of such a call are unspecified).
 *   - new_tokens of 2^28 - 16 and more are UNSUPPORTED, as is a max_context of 2^30.
 *   - context_lens (optional, may alias start_positions) receives
 *     start_positions[b] + new_tokens for every sequence that was written.
 */
typedef struct reef_kv_append_params {
    int64_t batch, kv_heads, head_dim; /* head_dim 64 or 128 */
    int64_t new_tokens;                /* tokens appended to every sequence */
    int64_t max_context;               /* capacity per sequence, a multiple of 16 */
} reef_kv_append_params;

reef_status reef_kv_append_int8(const reef_kv_append_params *p, const float *k_new,
                                const reef_strides *k_strides, const float *v_new,
                                const reef_strides *v_strides, const int32_t *start_positions,
                                int8_t *k_cache, int8_t *v_cache, float *k_scales,
                                float *v_scales, int32_t *context_lens, uint32_t *status_word,
                                hipStream_t stream);

/* The same into the paged layout; max_context <= max_blocks_per_seq * 16. */
reef_status reef_kv_append_int8_paged(const reef_kv_append_params *p, const float *k_new,
                                      const reef_strides *k_strides, const float *v_new,
                                      const reef_strides *v_strides,
                                      const int32_t *start_positions, const int32_t *block_table,
                                      int64_t max_blocks_per_seq, int64_t num_pages,
                                      int8_t *k_pages, int8_t *v_pages, float *k_scale_pages,
                                      float *v_scale_pages, int32_t *context_lens,
                                      uint32_t *status_word, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * The cache held in 4 bits: half the bytes of the int8 cache for a decode step to read. The
 * rule is quantize_rows' (quant.hpp:112-133) with 7 for 127: scale = max|x| / 7 of a token's
 * row (1 when max is 0), code = clamp(nearbyint(x / scale), -7, 7), IEEE division, ties to
 * even. A code c is stored as the nibble c + 8. The layouts are the int8 cache's with these
 * rows and pages:
 *   keys: a row is D/2 bytes; byte j holds channel j in its low nibble, channel j + D/2 in
 *   its high one.
 *   values: a page is [D, 8] bytes, a channel's 16 tokens in 8; token t's code is nibble
 *   8 (t / 8) + (t % 8) / 2 + 4 (t % 2) of them, low nibbles first (two tokens of an 8-token
 *   half lie 16 bits apart, so that one mask takes both).
 *   contiguous: k_cache [B, Hkv, L, D/2]; v_cache [B, Hkv, L/16, D, 8]; scales [B, Hkv, L].
 *   paged:      k_pages [P, Hkv, 16, D/2]; v_pages [P, Hkv, D, 8]; scales [P, Hkv, 16].
 * In all calls of this section block_table NULL means the contiguous cache of
 * p->max_context tokens a sequence (max_blocks_per_seq and num_pages are not used), otherwise
 * the paged one with max_context <= max_blocks_per_seq * 16. The int8 cache's page calls
 * (free, fork, reserve, compact) serve either pool. Decode and unpack take their scales on 16
 * bytes (unpack's keys': 4), as any allocation is.
 */

/* reef_kv_append_int8 (its limits, status bits and context_lens) into the 4-bit cache. The
 * codes beside the new ones, in the same bytes too, are left as they were. */
reef_status reef_kv_append_int4(const reef_kv_append_params *p, const float *k_new,
                                const reef_strides *k_strides, const float *v_new,
                                const reef_strides *v_strides, const int32_t *start_positions,
                                const int32_t *block_table, int64_t max_blocks_per_seq,
                                int64_t num_pages, uint8_t *k_cache, uint8_t *v_cache,
                                float *k_scales, float *v_scales, int32_t *context_lens,
                                uint32_t *status_word, hipStream_t stream);

/* `pages` pages of one head each, in memory order (a contiguous cache has B * Hkv * L / 16, a
 * pool P * Hkv), as fp32 rows: k and v [pages, 16, D], x = float(code) * scale. k or v NULL:
 * left out (its codes and scales then are not read). head_dim 64 or 128; pointers 16-byte
 * aligned, k_scales 4. */
reef_status reef_kv_unpack_int4(const uint8_t *k_pages, const uint8_t *v_pages,
                                const float *k_scales, const float *v_scales, int64_t pages,
                                int64_t head_dim, float *k, float *v, hipStream_t stream);

/* reef_kv_copy_pages for a pool of the 4-bit cache. */
reef_status reef_kv_copy_pages_int4(const int32_t *src, const int32_t *dst, int64_t n,
                                    int64_t kv_heads, int64_t head_dim, uint8_t *k_pages,
                                    uint8_t *v_pages, float *k_scale_pages, float *v_scale_pages,
                                    int64_t num_pages, uint32_t *status_word, hipStream_t stream);

/* The pages of 16 tokens that a decode step reads, for every (sequence, kv head): the first
 * counts[b][h] entries of pages[b][h], numbers of the sequence's pages (page i holds tokens
 * 16 i .. 16 i + 15), in any order. A negative entry is left out, one at or past the
 * sequence's ceil(len / 16) sets BAD_PAGE and is left out; a page listed twice counts twice.
 * A count outside [0, max_pages] sets BAD_LENGTH and yields zeros, as does 0 (without a bit). */
typedef struct reef_page_selection {
    const int32_t *pages;  /* [B, Hkv, max_pages], on the device */
    const int32_t *counts; /* [B, Hkv], on the device */
    int64_t max_pages;     /* below 2^26 */
} reef_page_selection;

/* The decode step of reef_attention_decode_int8 over the 4-bit cache, over all keys
 * (selection NULL) or the listed pages' alone. context_lens may be NULL for the contiguous
 * cache without a selection. The workspace is the int8 decode's, of the same size. With a
 * window, tokens before it take no part, whatever is listed. */
reef_status reef_attention_decode_int4(const reef_decode_params *p, const int8_t *q,
                                       const float *q_scales, const uint8_t *k_cache,
                                       const uint8_t *v_cache, const float *k_scales,
                                       const float *v_scales, const int32_t *block_table,
                                       int64_t max_blocks_per_seq, int64_t num_pages,
                                       const int32_t *context_lens,
                                       const reef_page_selection *selection, float *out,
                                       void *workspace, size_t workspace_bytes,
                                       uint32_t *status_word, hipStream_t stream);

/* reef_attention_prefill_int8_cache over the 4-bit cache (max_context as there; the workspace
 * is that call's, of the same size, zero-filled once). A long chunk's codes are widened on
 * their way into the workspace: the results of that call on an int8 cache of the same codes. A
 * short one, with REEF_ATTN_SCHED_AUTO and scales on 16 bytes, reads the cache in place as
 * decode does: the same sums in another order, with P in two fp16 parts. Either way a page number
 * outside [0, num_pages) sets BAD_PAGE and its page reads as zero codes; a short chunk looks at
 * the pages that its rows see. */
reef_status reef_attention_prefill_int4_cache(
    const reef_attention_params *p, const int8_t *q, const reef_strides *q_strides,
    const float *q_scales, const uint8_t *k_cache, const uint8_t *v_cache, const float *k_scales,
    const float *v_scales, int64_t max_context, const int32_t *block_table,
    int64_t max_blocks_per_seq, int64_t num_pages, float *out, const reef_strides *out_strides,
    void *workspace, size_t workspace_bytes, uint32_t *status_word, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Attention over the pages that a query selects, for caches too long to be read at every
 * step. Of every page the largest and the least key of each channel are kept; a query's
 * products with them bound its score with every key of the page, at 1/16 of the int8 keys'
 * and values' bytes. block_table NULL: contiguous, as in the section above.
 *
 * bounds: int8 codes [B, Hkv, L/16, 2, D] (contiguous) or [P, Hkv, 2, D] (paged), on 16 bytes;
 * bound_scales: one scale a page and head, [B, Hkv, L/16] or [P, Hkv].
 */

/* The bounds of the pages that positions start_positions[b] .. start_positions[b] +
 * new_tokens - 1 fall in, over those pages' tokens before start_positions[b] + new_tokens:
 * after an append, with its start positions (a page's earlier tokens are read again: the page
 * that reef_kv_reserve gave instead of a shared one, its tokens copied, needs nothing else);
 * after reef_kv_keep_int8, with the drafted tokens' start positions and number (rows that were
 * not kept only loosen their page's bounds). Pages that move take no bounds with them: after a
 * compaction and its copies, the _ragged call below. Of the keys x = float(code) * scale:
 * S = max|x| / 127 (1 where that is 0), [0][d] = min(127, ceil(max x_d / S)), [1][d] =
 * max(-127, floor(min x_d / S)), IEEE divisions. Key scales are positive and finite, as the
 * quantizers make them. Sizes and status bits as for reef_kv_append_int8 (a range past
 * max_context sets CAPACITY and writes nothing). */
reef_status reef_kv_page_bounds_int8(const reef_kv_append_params *p,
                                     const int32_t *start_positions, const int8_t *k_cache,
                                     const float *k_scales, const int32_t *block_table,
                                     int64_t max_blocks_per_seq, int64_t num_pages, int8_t *bounds,
                                     float *bound_scales, uint32_t *status_word,
                                     hipStream_t stream);

reef_status reef_kv_page_bounds_int4(const reef_kv_append_params *p,
                                     const int32_t *start_positions, const uint8_t *k_cache,
                                     const float *k_scales, const int32_t *block_table,
                                     int64_t max_blocks_per_seq, int64_t num_pages, int8_t *bounds,
                                     float *bound_scales, uint32_t *status_word,
                                     hipStream_t stream);

/* The same with an end for each sequence: the positions start_positions[b] ..
 * min(start_positions[b] + new_tokens, context_lens[b]) - 1, over those pages' tokens before
 * that end (context_lens [B] on the device; a sequence that ends at its start or before has
 * none, a length outside [0, max_context] sets BAD_LENGTH and writes nothing for it; a page
 * that several sequences name holds as many tokens of each, as forks' pages do). Starts of 0
 * and max_context tokens are every page that the sequences have tokens in. */
reef_status reef_kv_page_bounds_int8_ragged(
    const reef_kv_append_params *p, const int32_t *start_positions, const int32_t *context_lens,
    const int8_t *k_cache, const float *k_scales, const int32_t *block_table,
    int64_t max_blocks_per_seq, int64_t num_pages, int8_t *bounds, float *bound_scales,
    uint32_t *status_word, hipStream_t stream);

reef_status reef_kv_page_bounds_int4_ragged(
    const reef_kv_append_params *p, const int32_t *start_positions, const int32_t *context_lens,
    const uint8_t *k_cache, const float *k_scales, const int32_t *block_table,
    int64_t max_blocks_per_seq, int64_t num_pages, int8_t *bounds, float *bound_scales,
    uint32_t *status_word, hipStream_t stream);

/* For every (sequence, kv head) the `budget` pages to read, shared by the group's query
 * heads, as a reef_page_selection holds them: ascending, -1 behind the last. The first
 * `sinks` and the last `recent` pages of the sequence are always among them (recent >= 1,
 * sinks + recent <= budget), then those of the largest score, ties to the lowest page; all
 * pages where the sequence has no more than `budget`. A page's score is the largest over the
 * group's query heads of float(sum_d max(q_d, 0) [0][d] + min(q_d, 0) [1][d]) * (s_q * S),
 * the sum in whole numbers, the two products rounded to fp32 each: the same pages on every
 * run. q and q_scales as for decode; p->window, softmax_scale and num_splits are not used. A
 * page number outside [0, num_pages) sets BAD_PAGE, and that page is not selected; a length
 * outside [1, max_context] sets BAD_LENGTH, its counts are 0. Scales are finite. Workspace:
 * 16-byte aligned, reef_kv_select_pages_workspace_bytes(p) bytes (0: invalid sizes); nothing in
 * it is kept, calls that may run at the same time need separate ones. At most 65535 (sequence,
 * kv head) pairs. */
size_t reef_kv_select_pages_workspace_bytes(const reef_decode_params *p);

reef_status reef_kv_select_pages(const reef_decode_params *p, const int8_t *q,
                                 const float *q_scales, const int8_t *bounds,
                                 const float *bound_scales, const int32_t *block_table,
                                 int64_t max_blocks_per_seq, int64_t num_pages,
                                 const int32_t *context_lens, int64_t budget, int64_t sinks,
                                 int64_t recent, int32_t *pages, int32_t *counts, void *workspace,
                                 size_t workspace_bytes, uint32_t *status_word,
                                 hipStream_t stream);

/* The decode step of reef_attention_decode_int8 over the listed pages alone
 * (reef_attention_decode_int4 takes the same list). */
reef_status reef_attention_decode_int8_selected(
    const reef_decode_params *p, const int8_t *q, const float *q_scales, const int8_t *k_cache,
    const int8_t *v_cache, const float *k_scales, const float *v_scales,
    const int32_t *block_table, int64_t max_blocks_per_seq, int64_t num_pages,
    const int32_t *context_lens, const reef_page_selection *selection, float *out,
    void *workspace, size_t workspace_bytes, uint32_t *status_word, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Pages of the paged cache. block_table [batch, max_blocks_per_seq] int32 names the page of
 * every 16-token block of a sequence, -1 where it has none; context_lens [batch] int32 its
 * tokens; page_refs [num_pages] int32 how many table entries name a page: 0 is a free page,
 * more than 1 a page that sequences share. All lie on the device, and the caller starts with
 * every entry -1 and every count 0. One table may serve the caches of many layers: these
 * calls keep the table and the counts and leave lists of (source, destination) pages, -1 in
 * both where there is nothing to copy, for reef_kv_copy_pages on each layer's pool. Free
 * pages are given out lowest first, in the order of the sequences and of their blocks.
 *   - A sequence or pair with a negative index is padding; one past the end sets BAD_LENGTH,
 *     as does a length below 0 or (fork) beyond the table; a page number at or past
 *     num_pages, or a page given back that page_refs does not count, sets BAD_PAGE. Neither
 *     is followed.
 *   - batch, n <= 65535.
 */

/* The listed sequences give their pages back: their entries become -1, their lengths 0. */
reef_status reef_kv_free(const int32_t *sequences, int64_t n, int32_t *block_table,
                         int64_t max_blocks_per_seq, int32_t *context_lens, int64_t batch,
                         int32_t *page_refs, int64_t num_pages, uint32_t *status_word,
                         hipStream_t stream);

/* children[i] becomes a copy of parents[i] that shares its pages (those that hold tokens;
 * the pages the child had are given back). A sequence may be the parent of many, a child at
 * most once and then no parent in the same call (the table is unspecified otherwise, the
 * counts still agree with it). */
reef_status reef_kv_fork(const int32_t *parents, const int32_t *children, int64_t n,
                         int32_t *block_table, int64_t max_blocks_per_seq, int32_t *context_lens,
                         int64_t batch, int32_t *page_refs, int64_t num_pages,
                         uint32_t *status_word, hipStream_t stream);

/* Room for new_tokens more tokens of every sequence (one of length 0 too), in pages of its
 * own: blocks that the tokens at context_lens[b] .. context_lens[b] + new_tokens - 1 fall in
 * and that have no page get one, and those whose page is shared get one instead of it; where
 * that page holds tokens already (the last, partial one), copy_src[b] and copy_dst[b] (both
 * [batch]) name the two. A sequence that would pass max_blocks_per_seq * 16 tokens keeps its
 * blocks and sets CAPACITY, as do the blocks for which no free page is left (the others are
 * served; with their copies made, the call may be repeated once there are), unless the others
 * left such a block its page alone. Every sharer of a page gets one; the page that none keeps
 * becomes free. Lengths are not changed. The workspace needs reef_kv_reserve_workspace_bytes bytes, of any contents. */
size_t reef_kv_reserve_workspace_bytes(int64_t batch, int64_t new_tokens);

reef_status reef_kv_reserve(int32_t *block_table, int64_t max_blocks_per_seq,
                            const int32_t *context_lens, int64_t batch, int64_t new_tokens,
                            int32_t *page_refs, int64_t num_pages, int32_t *copy_src,
                            int32_t *copy_dst, void *workspace, size_t workspace_bytes,
                            uint32_t *status_word, hipStream_t stream);

/* The pool's live pages move to its front: with L of them, the k-th live page from the
 * pool's end that lies at or past L takes the k-th free place before L. The table and the
 * counts are rewritten; copy_src and copy_dst (num_pages / 2 entries each) list the moves,
 * all from pages at or past L to pages before it; num_live (NULL allowed) receives L. The
 * workspace needs reef_kv_compact_workspace_bytes bytes, of any contents. */
size_t reef_kv_compact_workspace_bytes(int64_t num_pages);

reef_status reef_kv_compact(int32_t *block_table, int64_t max_blocks_per_seq, int64_t batch,
                            int32_t *page_refs, int64_t num_pages, int32_t *copy_src,
                            int32_t *copy_dst, int32_t *num_live, void *workspace,
                            size_t workspace_bytes, uint32_t *status_word, hipStream_t stream);

/* Page src[i] of one layer's pool (keys, values and their scales, the paged layout above)
 * is copied to page dst[i], for n pairs. A pair with a negative page, or with both the same,
 * is left out; one past num_pages sets BAD_PAGE and is left out. No page may be a
 * destination twice, or a destination and a source (its contents are unspecified then). */
reef_status reef_kv_copy_pages(const int32_t *src, const int32_t *dst, int64_t n,
                               int64_t kv_heads, int64_t head_dim, int8_t *k_pages,
                               int8_t *v_pages, float *k_scale_pages, float *v_scale_pages,
                               int64_t num_pages, uint32_t *status_word, hipStream_t stream);

/* Of a sequence's last p->new_tokens tokens (drafted ones, appended before), the accepted
 * ones stay: rows kept[b][0 .. kept_lens[b] - 1] of them, ascending, move to the first
 * kept_lens[b] of their places, keys, values and scales. kept: [batch, new_tokens] int32
 * (entries past kept_lens[b] are not read); context_lens: [batch] int32, the drafted tokens
 * counted in; new_lens (optional, apart from context_lens, kept and kept_lens:
 * REEF_INVALID_ARGUMENT where it overlaps one) receives context_lens[b] - new_tokens +
 * kept_lens[b]. new_tokens <= 64. The rows behind the kept ones are left as they were. A length outside [new_tokens, max_context], a
 * kept_lens outside [0, new_tokens], or rows that are not ascending in [0, new_tokens) set
 * BAD_LENGTH, a page number outside [0, num_pages) BAD_PAGE; that sequence stays as it is
 * and new_lens[b] is its length. In the paged cache the drafted tokens' pages must be the
 * sequence's own (reef_kv_reserve). */
reef_status reef_kv_keep_int8(const reef_kv_append_params *p, const int32_t *kept,
                              const int32_t *kept_lens, const int32_t *context_lens,
                              int8_t *k_cache, int8_t *v_cache, float *k_scales, float *v_scales,
                              int32_t *new_lens, uint32_t *status_word, hipStream_t stream);

reef_status reef_kv_keep_int8_paged(const reef_kv_append_params *p, const int32_t *kept,
                                    const int32_t *kept_lens, const int32_t *context_lens,
                                    const int32_t *block_table, int64_t max_blocks_per_seq,
                                    int64_t num_pages, int8_t *k_pages, int8_t *v_pages,
                                    float *k_scale_pages, float *v_scale_pages,
                                    int32_t *new_lens, uint32_t *status_word, hipStream_t stream);

/* ---------------------------------------------------------------------------
 * Prefill over the int8 cache (chunked and multi-turn prompts): Attention::forward
 * with query_len > 1 on a cache that already holds the chunk's keys and values
 * (the engine appends first, then runs context() over every cached key with
 * query_start = key_len - query_len, attention.hpp:354-372 and :415). The cache is
 * the decode format above: contiguous when block_table is NULL (k_cache
 * [B, Hkv, max_context, D], v_cache [B, Hkv, max_context/16, D, 16], scales
 * [B, Hkv, max_context]), paged otherwise (k_cache [P, Hkv, 16, D], v_cache
 * [P, Hkv, D, 16], scales [P, Hkv, 16], block_table [B, max_blocks_per_seq],
 * P = num_pages; max_context is not used). p->kv_len is the number of cached
 * tokens of every sequence (the chunk's included, below 2^28), p->q_len the chunk length,
 * p->query_start normally kv_len - q_len; p->kv_granularity must be
 * REEF_SCALE_PER_TOKEN (the cache's scales). q, q_scales, out and out_strides are
 * as for reef_attention_prefill_int8. The call gathers the kv_len cached tokens of
 * every (sequence, kv head) into token-major rows in the workspace (at least
 * reef_attention_prefill_cache_workspace_bytes(p) bytes, 256-byte aligned; its
 * first part is the prefill's balanced-schedule workspace, so it must be
 * zero-filled before its first use, and every call leaves it ready for the next)
 * and runs the prefill attention over them. A page number outside [0, num_pages)
 * sets BAD_PAGE in status_word (optional) and reads as zero codes. */
size_t reef_attention_prefill_cache_workspace_bytes(const reef_attention_params *p);

reef_status reef_attention_prefill_int8_cache(
    const reef_attention_params *p, const int8_t *q, const reef_strides *q_strides,
    const float *q_scales, const int8_t *k_cache, const int8_t *v_cache, const float *k_scales,
    const float *v_scales, int64_t max_context, const int32_t *block_table,
    int64_t max_blocks_per_seq, int64_t num_pages, float *out, const reef_strides *out_strides,
    void *workspace, size_t workspace_bytes, uint32_t *status_word, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* REEF_HIP_ATTENTION_H */
