/*
 * siliconed_lm.h -- the operators of a decoder layer beside its 8-bit linears, for B200 (sm_100a):
 * libsiliconed_lm.so.
 *
 * The text encoders and prompt writers in front of Siliconed's DiTs decode token by token
 * (Sources/Siliconed/TextEncoder.swift, Qwen3VLDecoder.swift).  These entry points carry one decoder
 * layer in 8 bits: the residual addition, RMS norm and quantization to e4m3 (sl_rms_norm_quantize), the
 * product of such codes with a weight quantized in blocks (sl_linear_block_fp8), the QK-norm, position
 * rotation and append to a paged key-value cache (sl_append_paged), and the attention of one new token per
 * sequence over that cache (sl_paged_attention).  The reference has the layer's parts on Metal in 16 and
 * 32 bits; the paged cache, the e4m3 cache and the block-scaled product have no counterpart in it.
 *
 * Conventions: device pointers, integer sizes, `stream` a cudaStream_t.  Every function is asynchronous on
 * `stream`, allocates nothing and returns SL_OK, SL_INVALID_ARG or SL_CUDA_ERROR.  bf16 values are raw
 * 16-bit words, e4m3 values (e4m3fn) raw bytes.  Values that only the device sees (page numbers, positions,
 * sequence numbers) are checked on the device: one out of range is skipped, never dereferenced, and
 * reported by sl_errors.  Zero rows, tokens or sequences are a no-op.
 */
#ifndef SILICONED_LM_H
#define SILICONED_LM_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define SL_API __attribute__((visibility("default")))
#else
#define SL_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

enum { SL_OK = 0, SL_INVALID_ARG = 1, SL_CUDA_ERROR = 4, SL_TIMEOUT = 5, SL_OUT_OF_RANGE = 10 };

/* Element types of a residual stream or an addend, of a cache, and of a product's output. */
enum { SL_BF16 = 0, SL_F32 = 1, SL_E4M3 = 2 };

/* The two orders of a rotated pair in a head of D values: (2i, 2i + 1), or (i, i + D / 2). */
enum { SL_PAIRS_ADJACENT = 0, SL_PAIRS_HALVES = 1 };

/* Values under one scale of the e4m3 formats here. */
#define SL_BLOCK 128

/*
 * z = x + delta in fp32; x_out = z rounded to x's type; y = z * rsqrt(mean(z^2) + eps) * weight; then every
 * block of 128 consecutive values of a row gets the scale s = max(max|y| / 448, 1e-30) and the codes
 * e4m3(y / s), nearest-even.  Both quotients are products with a reciprocal: s is within an ulp of fp32 of its
 * definition, and what is rounded to a code within two of y / s, so that one code in many thousands, of a value
 * that lies on the middle between two codes, is the other one of the two.  The norm sees z before it is rounded
 * to x's type.  A block that holds a NaN or an infinity has that NaN or infinity as its scale, so that all of it
 * is NaN or infinite to a product.
 * x, x_out [rows, d] of x_type, delta [rows, d] of delta_type (SL_BF16 or SL_F32), weight fp32 [d] (NULL: 1),
 * codes bytes [rows, d], scales fp32 [rows, ceil(d / 128)].  x_out may be x.  delta NULL: z = x, and x_out
 * must be x or NULL (nothing is written to it).  norm 0: y = z * weight, the quantization alone (eps unused).
 * d a multiple of 16, at most 16384; x, x_out, delta, weight and codes 16-byte aligned.
 */
SL_API int sl_rms_norm_quantize(const void* x, int x_type, const void* delta, int delta_type, const float* weight,
                                float eps, int norm, int64_t rows, int d, void* x_out, uint8_t* codes, float* scales,
                                void* stream);

/*
 * New tokens into a paged cache.  qkv bf16 [tokens, (heads + 2 kv_heads) * head_dim] (q | k | v per token).
 * q and k heads: v * rsqrt(mean(v^2) + eps) * norm over the head when norm_q / norm_k (fp32 [head_dim]) are
 * given, then every pair rotated by (cos, sin) = freqs[position], freqs fp32 [max_pos, head_dim / 2, 2].
 * q bf16 [tokens, heads, head_dim].  Token i belongs to sequence seq[i] (NULL: i) at positions[i]; its key and
 * value go to slot position % page_size of page table[seq][position / page_size], table int32
 * [seqs, table_width].  The caches are [pages, kv_heads, page_size, head_dim]: bf16, or e4m3 with fp32 scales
 * [pages, kv_heads, page_size], s = max(max|v| / 448, 1e-30) over the head's values and codes e4m3(v / s), its
 * quotients as above (k_scale and v_scale NULL for a bf16 cache).  A token with a negative position is padding: its
 * q is written as zeros and nothing is appended; so is that of a position past max_pos, which is reported.  No two
 * tokens of a call share a slot.  head_dim 64 or 128; all tensors contiguous, 16-byte aligned.
 */
SL_API int sl_append_paged(const uint16_t* qkv, int64_t tokens, int heads, int kv_heads, int head_dim,
                           const float* norm_q, const float* norm_k, float eps, const float* freqs, int max_pos,
                           int pairs, const int32_t* seq, const int32_t* positions, const int32_t* table, int seqs,
                           int table_width, int64_t pages, int page_size, int cache_type, void* k_cache, void* v_cache,
                           float* k_scale, float* v_scale, uint16_t* q, void* stream);

/*
 * out[b, h] = sum_t p_t v_t / sum_t p_t with p_t = exp(scale q[b, h] . k_t - m) over the tokens t <
 * lengths[b] of sequence b, read through the page table from the caches that sl_append_paged fills; query head
 * h reads key-value head h / (heads / kv_heads).  q, out bf16 [batch, heads, head_dim]; lse fp32 [batch,
 * heads] (NULL: not wanted) gets log sum_t exp(scale q . k_t).  A sequence of length 0 (or whose scores are
 * all -inf, with finite values) gives zeros and lse -inf; a score of +inf gives NaN and lse +inf.  Slots past a
 * sequence's length are not read.  Scores, softmax statistics and sums are fp32.  For the product with v, p is held
 * to 16 bits (two bf16 terms); with an e4m3 cache p times its token's scale of v is rounded to f16, relative to the
 * largest such scale of the context so far: a term below 2^-29 of that scale has fewer than f16's 11 bits, one below
 * 2^-40 none.
 * head_dim 64 or 128; kv_heads divides heads.  The workspace (sl_paged_attention_workspace bytes, 16-byte
 * aligned) must be zero before its first use; every call leaves it ready for the next one.  Calls that may run
 * at the same time need workspaces of their own.
 */
SL_API int sl_paged_attention_workspace(int heads, int kv_heads, int head_dim, size_t* bytes);
SL_API int sl_paged_attention(const uint16_t* q, const void* k_cache, const void* v_cache, const float* k_scale,
                              const float* v_scale, int cache_type, const int32_t* table, const int32_t* lengths,
                              int batch, int heads, int kv_heads, int head_dim, int table_width, int64_t pages,
                              int page_size, float scale, uint16_t* out, float* lse, void* workspace,
                              size_t workspace_bytes, void* stream);

/*
 * y[i, j] = sum over blocks b of 128 along K of a_scales[i, b] * w_scales[j / 128, b] * (a[i, b] . w[j, b]),
 * + bias[j] when given: the product of e4m3 activations (sl_rms_norm_quantize's codes and scales) with a
 * published [N, K] e4m3 weight that has one fp32 scale per 128 x 128 block.  Each block's dot product is
 * accumulated in fp32 on the tensor cores and multiplied by its scales in fp32 before the sum over blocks.
 * a bytes [m, k], a_scales fp32 [m, ceil(k / 128)], w bytes [n, k], w_scales fp32 [ceil(n / 128),
 * ceil(k / 128)], bias bf16 [n] or NULL, y [m, n] bf16 or fp32 (y_type).  k a multiple of 16; a, w and y
 * 16-byte aligned.
 */
SL_API int sl_linear_block_fp8(const uint8_t* a, const float* a_scales, const uint8_t* w, const float* w_scales,
                               const uint16_t* bias, int64_t m, int64_t n, int64_t k, void* y, int y_type,
                               void* stream);

/*
 * The same calls with their arguments in a struct, in the same order.  For callers to whom each argument of a foreign call
 * costs: ctypes takes 2.7 us for 24 arguments, 0.7 us to pack and pass them at once.
 */
typedef struct {
  const void* x;
  int x_type;
  const void* delta;
  int delta_type;
  const float* weight;
  float eps;
  int norm;
  int64_t rows;
  int d;
  void* x_out;
  uint8_t* codes;
  float* scales;
  void* stream;
} sl_rms_norm_quantize_args;
SL_API int sl_rms_norm_quantize_with(const sl_rms_norm_quantize_args* args);

typedef struct {
  const uint16_t* qkv;
  int64_t tokens;
  int heads, kv_heads, head_dim;
  const float *norm_q, *norm_k;
  float eps;
  const float* freqs;
  int max_pos, pairs;
  const int32_t *seq, *positions, *table;
  int seqs, table_width;
  int64_t pages;
  int page_size, cache_type;
  void *k_cache, *v_cache;
  float *k_scale, *v_scale;
  uint16_t* q;
  void* stream;
} sl_append_paged_args;
SL_API int sl_append_paged_with(const sl_append_paged_args* args);

typedef struct {
  const uint16_t* q;
  const void *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  int cache_type;
  const int32_t *table, *lengths;
  int batch, heads, kv_heads, head_dim, table_width;
  int64_t pages;
  int page_size;
  float scale;
  uint16_t* out;
  float* lse;
  void* workspace;
  size_t workspace_bytes;
  void* stream;
} sl_paged_attention_args;
SL_API int sl_paged_attention_with(const sl_paged_attention_args* args);

typedef struct {
  const uint8_t* a;
  const float* a_scales;
  const uint8_t* w;
  const float* w_scales;
  const uint16_t* bias;
  int64_t m, n, k;
  void* y;
  int y_type;
  void* stream;
} sl_linear_block_fp8_args;
SL_API int sl_linear_block_fp8_with(const sl_linear_block_fp8_args* args);

/* Waits for the device, then reads and clears the library's error word on the current device: SL_TIMEOUT when a
 * bounded device-side wait gave up, SL_OUT_OF_RANGE when a page, position or sequence number was out of range
 * (the place in *site, which may be NULL), SL_CUDA_ERROR on an asynchronous CUDA error, else SL_OK. */
SL_API int sl_errors(int* site);

#ifdef __cplusplus
}
#endif

#endif /* SILICONED_LM_H */
