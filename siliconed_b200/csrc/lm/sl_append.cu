// New tokens into the paged key-value cache (sl_append_paged): QK-norm over each head, the rotation of pairs by
// the token's (cos, sin), q written for the attention, k and v written to their page slots as bf16 or as e4m3
// with one scale per token and head.
//
// Bound by HBM for prompts (each value is read and written once) and by latency for single tokens.  A group of
// head_dim / 8 lanes takes one head of one token, 16 bytes a lane; the norm's sum and the maximum stay inside the
// group, and the partner of a pair split over the two halves of the head is one shuffle away.
#include "sl_common.cuh"

namespace sl {
namespace {

struct Append {
  const uint16_t* qkv;
  int64_t tokens;
  int heads, kv_heads;
  const float *norm_q, *norm_k, *freqs;
  float eps;
  int max_pos;
  const int32_t *seq, *positions, *table;
  int seqs, table_width;
  int64_t pages;
  int page_size;
  void *k_cache, *v_cache;
  float *k_scale, *v_scale;
  uint16_t* q;
  int* err;
};

constexpr int kThreads = 256;

template <int kDim, bool kHalves, bool kE4m3>
__global__ void __launch_bounds__(kThreads) append_paged_k(const Append a) {
  constexpr int kLanes = kDim / 8;
  constexpr int kHalf = kDim / 2;
  sc::pdl_launch_dependents();
  sc::pdl_wait();
  const int all = a.heads + 2 * a.kv_heads;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
  const bool live = item < a.tokens * all;
  const int64_t token = live ? item / all : 0;
  const int head = live ? static_cast<int>(item % all) : 0;
  const int l = threadIdx.x % kLanes;
  const bool is_q = head < a.heads, is_v = head >= a.heads + a.kv_heads;
  int pos = live ? a.positions[token] : -1;
  if (pos >= a.max_pos) {
    sc::record_error(a.err, kErrRange, kSiteAppendPosition);
    pos = -1;
  }
  // The slot of a key or value head, -1 where nothing is to be written.
  int64_t slot = -1;
  if (pos >= 0 && !is_q) {
    const int s = a.seq != nullptr ? a.seq[token] : static_cast<int>(token);
    const int index = pos / a.page_size;
    if (s < 0 || s >= a.seqs) {
      sc::record_error(a.err, kErrRange, kSiteAppendSequence);
    } else if (index >= a.table_width) {
      sc::record_error(a.err, kErrRange, kSiteAppendPosition);
    } else {
      const int page = a.table[static_cast<int64_t>(s) * a.table_width + index];
      if (page < 0 || page >= a.pages)
        sc::record_error(a.err, kErrRange, kSiteAppendPage);
      else
        slot = (page * static_cast<int64_t>(a.kv_heads) + (head - a.heads) % a.kv_heads) * a.page_size + pos % a.page_size;
    }
  }
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (pos >= 0) {
    raw = reinterpret_cast<const uint4*>(a.qkv + (token * all + head) * kDim)[l];
    unpack8(raw, v);
  }
  // Every lane of the warp takes part in the shuffles, whatever its head is.
  const float* norm = is_q ? a.norm_q : a.norm_k;
  float ss = 0.0f;
#pragma unroll
  for (int t = 0; t < 8; ++t) ss += v[t] * v[t];
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, off);
  if (norm != nullptr && !is_v) {
    const float inv = 1.0f / sqrtf(ss / static_cast<float>(kDim) + a.eps);
    float w[8];
    load8(norm + 8 * l, w);
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = v[t] * inv * w[t];
  }
  if (kHalves) {
    float other[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) other[t] = __shfl_xor_sync(0xFFFFFFFFu, v[t], kLanes / 2);
    if (!is_v && pos >= 0) {
      const float* cs = a.freqs + (static_cast<int64_t>(pos) * kHalf + 8 * (l % (kLanes / 2))) * 2;
      const bool second = l >= kLanes / 2;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float4 f = reinterpret_cast<const float4*>(cs)[t];  // pairs 2t and 2t + 1
        v[2 * t] = second ? other[2 * t] * f.y + v[2 * t] * f.x : v[2 * t] * f.x - other[2 * t] * f.y;
        v[2 * t + 1] = second ? other[2 * t + 1] * f.w + v[2 * t + 1] * f.z : v[2 * t + 1] * f.z - other[2 * t + 1] * f.w;
      }
    }
  } else if (!is_v && pos >= 0) {
    const float* cs = a.freqs + static_cast<int64_t>(pos) * kDim + 8 * l;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float4 f = reinterpret_cast<const float4*>(cs)[t];
      const float e0 = v[4 * t], e1 = v[4 * t + 1], e2 = v[4 * t + 2], e3 = v[4 * t + 3];
      v[4 * t] = e0 * f.x - e1 * f.y;
      v[4 * t + 1] = e0 * f.y + e1 * f.x;
      v[4 * t + 2] = e2 * f.z - e3 * f.w;
      v[4 * t + 3] = e2 * f.w + e3 * f.z;
    }
  }
  uint32_t m = 0;
  if (kE4m3) {
    m = abs_max8(v);
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
  }
  if (!live) return;
  if (is_q) {
    reinterpret_cast<uint4*>(a.q + (token * a.heads + head) * kDim)[l] = pack8(v);
  } else if (slot >= 0) {
    if (kE4m3) {
      const float s = scale_of(m);
      reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_v ? a.v_cache : a.k_cache) + slot * kDim)[l] = quantize8(v, s);
      if (l == 0) (is_v ? a.v_scale : a.k_scale)[slot] = s;
    } else {
      reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_v ? a.v_cache : a.k_cache) + slot * kDim)[l] =
          is_v ? raw : pack8(v);
    }
  }
}

template <int kDim>
cudaError_t launch_append(const Append& a, bool halves, bool e4m3, cudaStream_t stream) {
  const int64_t per = kThreads / (kDim / 8);
  const int64_t grid = (a.tokens * (a.heads + 2 * a.kv_heads) + per - 1) / per;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  auto kernel = halves ? (e4m3 ? append_paged_k<kDim, true, true> : append_paged_k<kDim, true, false>)
                       : (e4m3 ? append_paged_k<kDim, false, true> : append_paged_k<kDim, false, false>);
  return launch(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, a);
}

}  // namespace
}  // namespace sl

extern "C" int sl_append_paged(const uint16_t* qkv, int64_t tokens, int heads, int kv_heads, int head_dim,
                               const float* norm_q, const float* norm_k, float eps, const float* freqs, int max_pos,
                               int pairs, const int32_t* seq, const int32_t* positions, const int32_t* table, int seqs,
                               int table_width, int64_t pages, int page_size, int cache_type, void* k_cache,
                               void* v_cache, float* k_scale, float* v_scale, uint16_t* q, void* stream) {
  using namespace sl;
  if (tokens < 0 || heads < 1 || kv_heads < 1 || heads > 65536 || kv_heads > 65536 ||
      (head_dim != 64 && head_dim != 128) || max_pos < 1 ||
      (pairs != SL_PAIRS_ADJACENT && pairs != SL_PAIRS_HALVES) || seqs < 1 || table_width < 1 || pages < 1 ||
      page_size < 1 || (cache_type != SL_BF16 && cache_type != SL_E4M3))
    return SL_INVALID_ARG;
  if (seq == nullptr && tokens > seqs) return SL_INVALID_ARG;
  if (tokens == 0) return SL_OK;
  for (const void* p : {static_cast<const void*>(qkv), static_cast<const void*>(freqs), static_cast<const void*>(k_cache),
                        static_cast<const void*>(v_cache), static_cast<const void*>(q)})
    if (p == nullptr || !aligned(p, 16)) return SL_INVALID_ARG;
  if (positions == nullptr || table == nullptr || !aligned(positions, 4) || !aligned(table, 4) || !aligned(seq, 4) ||
      !aligned(norm_q, 16) || !aligned(norm_k, 16))
    return SL_INVALID_ARG;
  const bool e4m3 = cache_type == SL_E4M3;
  if (e4m3 != (k_scale != nullptr) || e4m3 != (v_scale != nullptr) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return SL_INVALID_ARG;
  int* const err = current_device().err;
  if (err == nullptr) return SL_CUDA_ERROR;
  const Append a{qkv,       tokens,  heads,  kv_heads, norm_q,      norm_k, freqs,     eps,     max_pos, seq,     positions,
                 table,     seqs,    table_width, pages, page_size, k_cache, v_cache, k_scale, v_scale, q,       err};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool halves = pairs == SL_PAIRS_HALVES;
  return status_of(head_dim == 64 ? launch_append<64>(a, halves, e4m3, st) : launch_append<128>(a, halves, e4m3, st));
}
