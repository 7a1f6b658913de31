/*
 * qlinear.h -- C ABI of libqlinear, the B200 (sm_100a) group-wise affine Q4/Q8
 * quantized-linear library.
 *
 * This ABI is the drop-in boundary for the reference's quantized-linear path.
 * The reference (SceneWorks/mlx-gen, Rust on MLX) reaches the arithmetic
 * through mlx-rs; each entry point below names the call it replaces.
 *
 * Conventions
 *   - Every pointer argument is caller-owned DEVICE memory (except ql_last_error's
 *     result).  The library allocates nothing on any call path.
 *   - Row-major, contiguous.  W is [N, K] (out, in), x is [M, K], y is [M, N].
 *   - Packing (byte-identical to MLX affine quantization): wq is uint32
 *     [N, K*bits/32]; element k of a row is code (wq[k/(32/bits)] >> (bits*(k%(32/bits))))
 *     & (2^bits-1); scales / biases are [N, K/group_size]; w = code*scale + bias.
 *   - `stream` is a cudaStream_t (NULL = legacy default stream).  Calls are
 *     asynchronous, hold no global mutable state and may run concurrently on
 *     different streams -- except ql_quantized_matmul_noalloc, whose LoRA calls share
 *     one fixed device array (see its declaration).
 *   - Return value is a ql_status.  On failure, ql_last_error() returns a
 *     thread-local message.  No call aborts or exits.
 */
#ifndef QLINEAR_H
#define QLINEAR_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    QL_F32 = 0,
    QL_BF16 = 1,
    QL_F16 = 2,
} ql_dtype;

typedef enum {
    QL_OK = 0,
    QL_EINVAL_SHAPE = 1,  /* K % group_size, sizes <= 0, mismatched shapes      */
    QL_EUNSUPPORTED = 2,  /* bits not in {4,8}, group_size not in {32,64,128},
                             dtype combination without a kernel                 */
    QL_ECUDA = 3,         /* a CUDA runtime / driver call failed                */
    QL_EINVAL_ARG = 4,    /* NULL pointer, misaligned pointer, small workspace  */
    QL_ETIMEOUT = 5,      /* a kernel's bounded wait ran out (see ql_device_error) */
} ql_status;

typedef enum {
    QL_ACT_NONE = 0,
    QL_ACT_GELU_TANH = 1, /* 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3)))     */
    QL_ACT_GELU_ERF = 2,  /* 0.5 x (1 + erf(x / sqrt 2))                         */
    QL_ACT_SWIGLU = 3,    /* silu(x W^T) * (x W_up^T); needs the *_up weights    */
} ql_act;

typedef enum {
    QL_KERNEL_AUTO = 0,    /* GEMV for M <= 8, tcgen05 GEMM otherwise (bf16)    */
    QL_KERNEL_GENERIC = 1, /* CUDA-core fp32 kernel; any dtype                   */
    QL_KERNEL_GEMV = 2,    /* M <= 8, bf16 x and bf16 scales                     */
    QL_KERNEL_GEMM = 3,    /* tcgen05 / TMEM GEMM, one CTA per MMA (cta_group::1) */
    QL_KERNEL_GEMM_PAIR = 4, /* the same GEMM on CTA pairs (cta_group::2); slower today */
    QL_KERNEL_GEMV_TC = 5, /* the tcgen05 GEMV alone (M <= 8, no LoRA, group 64/128 or Q8/32;
                              QL_EUNSUPPORTED otherwise); QL_KERNEL_GEMV picks it for wide N */
    QL_KERNEL_GEMV_TMA = 6, /* the TMA-fed mma.sync GEMV alone (M <= 8, K a whole number of
                               8-group batches)                                          */
    QL_KERNEL_GEMV_REGS = 7, /* the register-fed GEMV alone (M <= 8)                     */
} ql_kernel;

typedef enum {
    QL_ROPE_HALF = 0,        /* pairs (i, i + rotary_dim / 2)                           */
    QL_ROPE_INTERLEAVED = 1, /* pairs (2i, 2i + 1)                                      */
} ql_rope_layout;

/* Fused epilogue and options of ql_quantized_matmul.  Zero-initialise, then set
 * what is needed.  Replaces the ops the reference runs after quantized_matmul:
 * the bias add (src/adapters.rs:318-320), the LoRA residual sum
 * (src/adapters.rs:260-270,545-547), GELU (src/nn.rs:321-355) and SwiGLU
 * (mlx-gen-z-image/src/feed_forward.rs:34-38). */
typedef struct {
    const void *bias;          /* [N] in y's dtype, or NULL                           */
    int act;                   /* ql_act                                               */
    /* SwiGLU second projection (w3 / "up"), same shapes and dtypes as the main one. */
    const uint32_t *wq_up;
    const void *scales_up;
    const void *biases_up;
    const void *bias_up;       /* [N] or NULL                                          */
    /* LoRA residual: y += lora_scale * (x . A) . B with A [K, rank], B [rank, N] in
     * x's dtype, any rank in [1, 4096].  Needs `workspace` of ql_matmul_workspace_size(). */
    const void *lora_a;
    const void *lora_b;
    int64_t lora_rank;
    float lora_scale;
    void *workspace;
    size_t workspace_bytes;
    int kernel;                /* ql_kernel (QL_KERNEL_AUTO unless testing a path)     */
    int max_ctas;              /* GEMM: cap on resident CTAs (0 = one per SM); leaves
                                  SMs free for a collective running alongside          */
    /* Gated residual (the DiT blocks' `x + gate * linear(x)`, src/nn.rs:166-176):
       y = residual + gate * f(x W^T + bias), each op rounded to y's dtype.  NULL residual:
       off.  gate [rows, N] with row m / gate_period (gate_period 0: one row for all M);
       NULL gate: y = residual + f(...).  Both in y's dtype; residual may alias y.      */
    const void *residual;      /* [M, N]                                               */
    const void *gate;          /* [M / gate_period, N] or [N]                          */
    int64_t gate_period;       /* token rows per gate row (0: one gate row)            */
    /* LoKr residual (src/adapters.rs:263-266): y += lokr_scale * x . delta^T, delta a dense
       [N, K] matrix in x's dtype (the reconstructed Kronecker product).  The tensor-core
       path adds lokr_scale * delta to each dequantized weight (no extra MMA); it needs
       the 1-CTA GEMM without SwiGLU (QL_KERNEL_AUTO picks it for any M).  NULL: off.  */
    const void *lokr_delta;
    float lokr_scale;
} ql_epilogue;

/* Library version (major*10000 + minor*100 + patch). */
int ql_version(void);

/* Thread-local message describing the last failure on this thread ("" if none). */
const char *ql_last_error(void);

/* Reads (and with clear != 0 resets) the device-side error word that kernels set
 * when a bounded wait runs out.  Synchronises the current device.  0 = no error. */
int ql_device_error(int clear);

/* Test hook for the failure path (no counterpart in the reference, whose failure model is
 * a cooperative cancel flag, gen-core/src/runtime.rs:239-258).  Every pipelined kernel's
 * waits are bounded: when one runs out the kernel records a DEV_ERR timeout code in the
 * device error word (read with ql_device_error), every role drains, TMEM is freed and the
 * kernel returns; the context stays usable.  wait_limit_ns replaces the 2 s limit on the
 * current device (0 restores it); flags bit 0 makes the tcgen05 GEMM's TMA producer issue
 * nothing, bit 1 the tcgen05 attention's, bit 2 makes that one stop half-way, so their consumers'
 * waits run out.  Synchronises the current device.  Not for
 * production use: set flags back to 0 afterwards. */
int ql_debug_inject(unsigned flags, unsigned long long wait_limit_ns);

/* Replaces mlx_rs::ops::quantize(w, group_size, bits) -> (wq, scales, biases)
 * (called at src/quant.rs:140, src/adapters.rs:533-537 via
 * QuantizedLinear::try_from_linear, src/nn.rs:91-93).  w [N, K] in w_dtype;
 * scales/biases written in sb_dtype (the reference stores them in w's dtype). */
int ql_quantize(const void *w, int w_dtype, int64_t N, int64_t K, int group_size, int bits,
                uint32_t *wq, void *scales, void *biases, int sb_dtype, void *stream);

/* Replaces mlx_rs::ops::dequantize(wq, scales, biases, group_size, bits)
 * (src/nn.rs:55, tests/quant_parity.rs:53).  out [N, K] in out_dtype;
 * w = fma(code, scale, bias) in fp32, rounded once. */
int ql_dequantize(const uint32_t *wq, const void *scales, const void *biases, int sb_dtype,
                  int64_t N, int64_t K, int group_size, int bits, void *out, int out_dtype,
                  void *stream);

/* Replaces the quantized TokenEmbedding gather: take_axis(wq|scales|biases, ids)
 * followed by dequantize and a cast (src/nn.rs:42-59).  ids [R] int64 into the
 * N rows; out [R, K] in out_dtype.  Each value is fma(code, scale, bias) in fp32
 * rounded to sb_dtype (dequantize's output dtype), then converted to out_dtype.  An id
 * outside [0, N) yields a zero row and sets the device error word. */
int ql_dequantize_rows(const int64_t *ids, int64_t R, const uint32_t *wq, const void *scales,
                       const void *biases, int sb_dtype, int64_t N, int64_t K, int group_size,
                       int bits, void *out, int out_dtype, void *stream);

/* The DiT blocks' adaLN prologue in one pass: y = (1 + scale) * layer_norm(x) + shift.
   Replaces mlx_rs::fast::layer_norm(x, None, None, eps) followed by nn::modulate
   (mlx-gen-flux/src/transformer.rs:891-913, src/nn.rs:262-287).  x bf16 [M, D], D a
   multiple of 8; scale / shift bf16 [M / period, D] (period 0: one row for all M) or NULL
   (plain layer norm).  y_dtype QL_BF16: each modulate op rounded to bf16 (FLUX.1, the 1
   in scale's dtype); QL_F32: computed and stored in f32 (FLUX.2, a strong f32 1). */
int ql_layernorm_modulate(const void *x, int64_t M, int64_t D, float eps, const void *scale, const void *shift,
                          int64_t period, void *y, int y_dtype, void *stream);

/* Replaces mlx_rs::ops::quantized_matmul(x, wq, scales, biases, transpose=true,
 * group_size, bits) as called by LinearBase::forward (src/adapters.rs:309-317),
 * plus the ops fused through `ep` (may be NULL).  y [M, N] in y_dtype.
 * transpose must be 1 (the only form the reference uses). */
int ql_quantized_matmul(const void *x, int x_dtype, int64_t M, int64_t K, const uint32_t *wq,
                        const void *scales, const void *biases, int sb_dtype, int64_t N,
                        int group_size, int bits, int transpose, const ql_epilogue *ep,
                        void *y, int y_dtype, void *stream);

/* Bytes of device workspace ql_quantized_matmul needs for this shape and
 * epilogue (0 when none; the LoRA residual needs M * round_up(rank, 64) * 2). */
size_t ql_matmul_workspace_size(int64_t M, int64_t N, int64_t K, const ql_epilogue *ep);

/* Workspace for ql_quantized_matmul when x is x_dtype: the LoRA need above, or -- for f32 /
 * f16 activations -- the two bf16 pieces of x ([M, 2 * round_up(K, 64)] bf16) that the
 * tensor-core path for those dtypes stages.  Given that workspace, an f32 / f16 x with bf16
 * or f16 scales, f32 / f16 y, a plain or GELU linear (no SwiGLU, LoRA, LoKr or gated
 * residual) runs on the tcgen05 GEMM in three bf16 passes (x and each dequantized weight
 * split into two bf16 pieces: about 16 significant bits per product, fp32 accumulation --
 * the activations of FLUX.2 / Qwen image streams / LTX text encoders, src/adapters.rs:252,
 * src/nn.rs:295); without it those calls run on the CUDA-core kernel. */
size_t ql_matmul_workspace_size_x(int64_t M, int64_t N, int64_t K, const ql_epilogue *ep, int x_dtype);

/* Same as ql_quantized_matmul, for callers that cannot allocate device memory
 * (allocator hooks, real-time loops that must not enter the driver's allocator,
 * runtimes whose memory is fully reserved).  No counterpart in the reference.
 * The LoRA workspace comes from a fixed 8 MiB device array inside the library
 * (ep->workspace is ignored); a request above that (M * round_up(rank, 64) * 2
 * bytes) returns QL_EUNSUPPORTED.  The first call on a device (LoRA or not) looks up the array
 * with that device current -- make it before any stream capture.  Calls share the
 * array: calls that overlap on the GPU race.  Allocates nothing. */
int ql_quantized_matmul_noalloc(const void *x, int x_dtype, int64_t M, int64_t K,
                                const uint32_t *wq, const void *scales, const void *biases,
                                int sb_dtype, int64_t N, int group_size, int bits, int transpose,
                                const ql_epilogue *ep, void *y, int y_dtype, void *stream);

/* ---- decoder operators: what stands between the quantized linears of a decoder layer or a
 * DiT block.  Pages: a cache of one layer is [num_pages, Hkv, page_size, D] for the keys and
 * the same for the values; page p starts page_stride elements after page p - 1 and its
 * [Hkv, page_size, D] are contiguous.  A sequence's page table row lists its pages in order;
 * position j is slot table[j / page_size] * page_size + j % page_size. */

/* The norms around a block, fused with its gate and residual scale:
 *     u = post_weight ? rms(y) * (weight_offset + post_weight) : y
 *     r_out = residual + alpha * gate * u
 *     h = rms(r) * (weight_offset + weight) * (1 + scale),   rms(x) = x / sqrt(mean(x^2) + eps)
 * in fp32, each output rounded once (h is computed from the unrounded r).  y, weights, gate,
 * scale and h in y_dtype, residual and r_out in r_dtype (y's, or f32).  D in [1, 32768];
 * y_stride / r_stride: elements between rows of y / residual (h and r_out are contiguous).
 * gate / scale: [rows, D] with row m / period (period 0: one row for all), or NULL; post_weight
 * may be NULL.  r_out may be residual itself (same stride), h may be y. */
int ql_norm_residual(const void *y, int y_dtype, int64_t y_stride, const void *residual, int r_dtype, int64_t r_stride,
                     int64_t M, int64_t D, const void *weight, float weight_offset, const void *post_weight,
                     const void *gate, int64_t gate_period, float alpha, const void *scale, int64_t scale_period,
                     float eps, void *h, void *r_out, void *stream);

/* Rotary positions: q [T, Hq, D] and k [T, Hk, D] (element strides given, D contiguous) ->
 * contiguous q_out, k_out.  (a, b) -> (a cos - b sin, b cos + a sin) on the pairs of the first
 * rotary_dim elements of each head, the rest copied; fp32, one rounding.  table: fp32
 * [table_rows, rotary_dim], row p holds position p's rotary_dim / 2 cosines, then its sines.
 * A position outside the table gives zeros and sets the device error word.  q_out may be q and
 * k_out k when those are contiguous.  Hq or Hk may be 0. */
int ql_rope(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k, int64_t k_token_stride,
            int64_t k_head_stride, int dtype, int64_t T, int Hq, int Hk, int D, int rotary_dim, int layout,
            const float *table, int64_t table_rows, const int64_t *positions, void *q_out, void *k_out, void *stream);

/* The same, with the rotated k and v written to the cache at slots[t] (page * page_size +
 * offset) instead of k_out.  A negative slot: the token is not cached (padding).  A slot past
 * the cache, or a bad position: not cached, device error word set.  Slots that are written must
 * be distinct.  page_size: a power of two. */
int ql_rope_append(const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *k, int64_t k_token_stride,
                   int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride, int dtype,
                   int64_t T, int Hq, int Hkv, int D, int rotary_dim, int layout, const float *table,
                   int64_t table_rows, const int64_t *positions, const int64_t *slots, void *k_cache, void *v_cache,
                   int64_t num_pages, int64_t page_stride, int page_size, void *q_out, void *stream);

/* Attention of each sequence's new tokens over its paged cache (the new tokens' keys and
 * values already appended): out = softmax(scale q k^T) v.  q [T, Hq, D] (strides given), out
 * [T, Hq, D] contiguous; q head h reads kv head h / (Hq / Hkv).  Sequence b's tokens are
 * q_starts[b] .. q_starts[b + 1] - 1 (q_starts [B + 1], covering 0 .. T), its cached positions
 * 0 .. kv_lens[b] - 1, its pages page_table[b * table_stride ..].  Token i of q_len stands at
 * p = kv_len - q_len + i and sees the positions j < kv_len, with causal j <= p, with window > 0
 * (needs causal) j > p - window.  A token that sees nothing gets zeros (so does one all of whose
 * scores are -inf); a NaN among a row's scores, or a score of +inf, makes the row NaN.  max_q / max_kv: upper
 * bounds of q_len / kv_len known to the host; a sequence beyond them, or a page index outside
 * the cache, sets the device error word (its output is unspecified).  Entries of the page table
 * and cache contents that no token of a sequence sees are not used.
 * dtype bf16 or f16; D 64, 96, 128 or 256; page_size a power of two in [16, 1024]; at most 65535
 * sequences; max_q * Hq / Hkv at most 16776960 (D 64, 128) or 2^30, max_kv at most 2^30; fp32
 * softmax, the weights rounded to dtype for the second product.  q and the caches 16-byte
 * aligned, q's strides multiples of 8; out and workspace (see below) 32-byte aligned. */
int ql_paged_attention(const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int64_t T, int Hq,
                       int Hkv, int D, const void *k_cache, const void *v_cache, int64_t num_pages,
                       int64_t page_stride, int page_size, const int32_t *page_table, int64_t table_stride,
                       const int32_t *q_starts, const int32_t *kv_lens, int64_t B, int64_t max_q, int64_t max_kv,
                       float scale, int causal, int64_t window, void *out, void *workspace, size_t workspace_bytes,
                       void *stream);

/* Bytes of device workspace ql_paged_attention needs for these sizes (0: none). */
size_t ql_paged_attention_workspace_size(int64_t T, int Hq, int Hkv, int D, int64_t B, int64_t max_q, int64_t max_kv,
                                         int64_t window);

/* The same, always causal, with the first `sinks` positions visible beside the window: token p sees
 * the positions j <= p with j > p - window or j < sinks.  sinks at most 1024, and 0 without a
 * window.  Pages between the sinks and the windows of a sequence's new tokens are not used (their
 * entries may be anything), so a sequence without end keeps a fixed number of pages.  The
 * workspace is ql_paged_attention_workspace_size's for that window. */
int ql_sink_attention(const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int64_t T, int Hq,
                      int Hkv, int D, const void *k_cache, const void *v_cache, int64_t num_pages, int64_t page_stride,
                      int page_size, const int32_t *page_table, int64_t table_stride, const int32_t *q_starts,
                      const int32_t *kv_lens, int64_t B, int64_t max_q, int64_t max_kv, float scale, int64_t window,
                      int64_t sinks, void *out, void *workspace, size_t workspace_bytes, void *stream);

/* The index tensors of a step in which sequence b gets new_tokens[b] tokens more than its
 * lengths[b]: kv_lens[b] = their sum, q_starts [B + 1] = exclusive sums of new_tokens, and for each
 * new token its position and its slot (page * page_size + offset, from page_table
 * [B, table_width] with rows table_stride entries apart), in the order of the sequences.  Rows behind
 * the last token, up to max_tokens, get position 0 and slot -1 (not cached).  With free_pages
 * [num_free] the pages that the new tokens need beyond those of the old ones are taken from it,
 * from entry taken[0] on in the order of the sequences, and entered in page_table; taken_out[0] =
 * taken[0] + their number.  Without (NULL) the tables hold every page already, taken and taken_out
 * are not used.  All or nothing: counts below 0, more tokens than max_tokens, pages past table_width or
 * past num_free give a step without tokens (kv_lens = lengths, q_starts 0, nothing taken) and set
 * the device error word; so does a negative table entry, whose tokens get slot -1.  kv_lens may be
 * lengths and taken_out taken: a captured call then advances the sequences at every replay; any other output over an
 * input, an output or the page table's rows is refused.
 * page_size: a power of two. */
int ql_plan_step(int32_t *page_table, int64_t table_stride, int64_t table_width, const int32_t *lengths,
                 const int32_t *new_tokens, int64_t B, int page_size, int64_t max_tokens, const int32_t *free_pages,
                 int64_t num_free, const int32_t *taken, int64_t *positions, int64_t *slots, int32_t *q_starts,
                 int32_t *kv_lens, int32_t *taken_out, void *stream);

/* The same, and a step after which a sequence would hold more than max_kv tokens has no room either: the bound that the
 * attention behind it was captured with, which a replay too many would pass inside its last page. */
int ql_plan_step_within(int32_t *page_table, int64_t table_stride, int64_t table_width, const int32_t *lengths,
                        const int32_t *new_tokens, int64_t B, int page_size, int64_t max_tokens, int64_t max_kv,
                        const int32_t *free_pages, int64_t num_free, const int32_t *taken, int64_t *positions,
                        int64_t *slots, int32_t *q_starts, int32_t *kv_lens, int32_t *taken_out, void *stream);

/* One token per row of logits [B, V] (row_stride elements between rows, 0: all the same) from random numbers u [B] in [0, 1):
 *     w_i = exp((x_i - max x) / temperature); in the order of x (descending, equal ones by index) the
 *     first top_k stay (0: all), of those the shortest prefix with a sum of at least top_p times
 *     theirs (one token at least; 1: all), of those the ones with w_i >= min_p;
 *     tokens[b] = the first that stays, by index, with (sum up to it) > u (sum of all that stay).
 * temperature 0: the largest logit, the lowest index of equal ones; others count as 2e-17 at least and 4e28
 * at most.  Each setting is one number for each row
 * (a pointer) or for all (NULL and the ..._all argument, kept in 64 bits).  Weights are computed in 64 bits and
 * summed as whole numbers (of 2^-46, for more than 2^17 tokens 2^(ceil(log2 V) - 63)), so that a row's token does not
 * depend on the rest of the batch, and one whose weight rounds to 0 is never drawn, not by u = 0 or 1 either; a logit of -inf is never drawn, those of +inf share everything.  u is taken as at
 * least 0, and 1 or more gives the last token that stays.  A row with a NaN (logits, settings or u), a
 * negative temperature or nothing above -inf: token -1, log-probability NaN.  logprobs [B] or
 * NULL: the logarithm of the probability with which the token was drawn (0 for temperature 0).
 * dtype f32, bf16 or f16, a row at most 1310208 bytes. */
int ql_sample(const void *logits, int dtype, int64_t row_stride, int64_t B, int64_t V, const float *u,
              const float *temperature, double temperature_all, const int32_t *top_k, int64_t top_k_all,
              const float *top_p, double top_p_all, const float *min_p, double min_p_all, int64_t *tokens,
              float *logprobs, void *stream);

/* Copies pages inside a pool: page dst[i] := page src[i] in each of `planes` planes (the keys or
 * values of one layer), plane_stride bytes apart, pages page_stride bytes apart, page_bytes each
 * (all multiples of 16).  src and dst are HOST arrays of n indices, read before the call
 * returns.  Every index must be inside num_pages, no page twice a destination, no destination a
 * source.  For a fork's copy on write and for compaction. */
int ql_copy_pages(void *pool, int64_t planes, int64_t plane_stride, int64_t num_pages, int64_t page_stride,
                  int64_t page_bytes, const int32_t *src, const int32_t *dst, int64_t n, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* QLINEAR_H */
