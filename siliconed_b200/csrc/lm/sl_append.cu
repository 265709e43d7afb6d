// New tokens into the paged key-value cache (sl_append_paged): QK-norm over each head, the rotation of pairs by
// the token's (cos, sin), q written for the attention, k and v written to their page slots as bf16 or as e4m3
// with one scale per token and head.
//
// Bound by latency: for single tokens a launch's, for prompts that of the dependent reads with which every CTA begins (the
// position, then the sequence and page, and the (cos, sin) of that position), three rounds of CTAs one after another for 2711
// tokens: issue slots are taken in 54 % of the cycles and waiting for loads is the first stall; 17 us where the bytes take 8.6.
// One CTA per token;
// groups of head_dim / 16 lanes take its heads in turns, three turns' loads at once, with the token's (cos, sin) and page
// slot loaded once.  A lane holds 8 values of a head's first half and the same 8 of its second half, so both orders of
// pairs rotate inside a lane, and the norm's sum and the maximum take three shuffles for 16 values.  (8 values a lane,
// the partner fetched by shuffles, IEEE divisions: 24 us for 2400 tokens of 42 heads where this takes 17.)
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

constexpr int kThreads = 128;
// Heads of a group on their way at once, and the CTAs an SM that the registers are held to: of 64 values a head eight (2400
// tokens of 20 heads 5.7 us, without 7.0); of 128 into an e4m3 cache six (a prompt's 2711 tokens 17.4 us, without 18.7, eight
// 20.8), into a bf16 cache none (2400 tokens of 48 heads 16.3 us, six 17.0).
template <int kDim>
constexpr int kTurns = kDim == 64 ? 2 : 3;
template <int kDim, bool kE4m3>
constexpr int kResident = kDim == 64 ? 8 : (kE4m3 ? 6 : 1);

template <int kDim, bool kHalves, bool kE4m3>
__global__ void __launch_bounds__(kThreads, kResident<kDim, kE4m3>) append_paged_k(const Append a) {
  constexpr int kLanes = kDim / 16, kGroups = kThreads / kLanes;
  constexpr int kHalf = kDim / 2;
  sc::pdl_launch_dependents();
  sc::pdl_wait();
  const int all = a.heads + 2 * a.kv_heads;
  const int64_t token = blockIdx.x;
  const int group = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
  // Of a head's 16-byte chunks: this lane's are l and l + kLanes.
  const uint4* src = reinterpret_cast<const uint4*>(a.qkv + token * all * kDim) + l;
  uint4 raw[kTurns<kDim>][2];
  const auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kTurns<kDim>; ++i) {
      const int head = first + i * kGroups + group;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        raw[i][h] = head < all ? src[(2 * head + h) * kLanes] : make_uint4(0, 0, 0, 0);
    }
  };
  load(0);
  int pos = a.positions[token];
  if (pos >= a.max_pos) {
    sc::record_error(a.err, kErrRange, kSiteAppendPosition);
    pos = -1;
  }
  // Where the token's keys and values go: the slot of key-value head 0, the next head's page_size further; -1: nowhere.
  int64_t slot = -1;
  if (pos >= 0) {
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
        slot = page * static_cast<int64_t>(a.kv_heads) * a.page_size + pos % a.page_size;
    }
  }
  // (cos, sin) of this lane's 8 pairs: of halves, pairs 8 l ..; adjacent, pairs 4 l .. + 3 and kDim / 4 + 4 l .. + 3.
  float2 cs[8];
  {
    const float4* f = reinterpret_cast<const float4*>(a.freqs + static_cast<int64_t>(max(pos, 0)) * kDim);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float4 v = f[kHalves ? 4 * l + t : (t < 2 ? 2 * l + t : kDim / 8 + 2 * l + t - 2)];
      cs[2 * t] = make_float2(v.x, v.y);
      cs[2 * t + 1] = make_float2(v.z, v.w);
    }
  }

  // Every lane of a warp takes part in the shuffles of every turn, whether its group has a head left or not.
  const auto work = [&](int first, int i) {
    const int head = first + i * kGroups + group;
    const bool live = head < all;
    const bool is_q = head < a.heads, is_v = head >= a.heads + a.kv_heads;
    float v[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (pos < 0) raw[i][h] = make_uint4(0, 0, 0, 0);
      unpack8(raw[i][h], v[h]);
    }
    const float* norm = is_q ? a.norm_q : a.norm_k;
    float ss = 0.0f;
#pragma unroll
    for (int t = 0; t < 8; ++t) ss += v[0][t] * v[0][t] + v[1][t] * v[1][t];
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, off);
    if (!is_v && pos >= 0) {  // padding stays zeros, whatever eps and the rotation table's first row are
      if (norm != nullptr) {
        const float inv = rsqrtf(ss * (1.0f / kDim) + a.eps);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float w[8];
          load8(norm + h * kHalf + 8 * l, w);
#pragma unroll
          for (int t = 0; t < 8; ++t) v[h][t] = v[h][t] * inv * w[t];
        }
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        float& x = kHalves ? v[0][t] : v[t / 4][t % 4 * 2];
        float& y = kHalves ? v[1][t] : v[t / 4][t % 4 * 2 + 1];
        const float e0 = x, e1 = y;
        x = e0 * cs[t].x - e1 * cs[t].y;
        y = e0 * cs[t].y + e1 * cs[t].x;
      }
    }
    uint32_t m = 0;
    if (kE4m3) {
      m = max(abs_max8(v[0]), abs_max8(v[1]));
#pragma unroll
      for (int off = kLanes / 2; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
    }
    if (live && is_q) {
      uint4* q = reinterpret_cast<uint4*>(a.q + (token * a.heads + head) * kDim) + l;
      q[0] = pack8(v[0]);
      q[kLanes] = pack8(v[1]);
    } else if (live && slot >= 0) {
      const int64_t to = slot + static_cast<int64_t>(head - a.heads - (is_v ? a.kv_heads : 0)) * a.page_size;
      if (kE4m3) {
        const float s = scale_of(m);
        uint2* c = reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_v ? a.v_cache : a.k_cache) + to * kDim) + l;
        c[0] = quantize8(v[0], s);
        c[kLanes] = quantize8(v[1], s);
        if (l == 0) (is_v ? a.v_scale : a.k_scale)[to] = s;
      } else {
        uint4* c = reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_v ? a.v_cache : a.k_cache) + to * kDim) + l;
        c[0] = is_v ? raw[i][0] : pack8(v[0]);
        c[kLanes] = is_v ? raw[i][1] : pack8(v[1]);
      }
    }
  };
#pragma unroll 1
  for (int first = 0; first < all; first += kTurns<kDim> * kGroups) {
    if (first != 0) load(first);
#pragma unroll
    for (int i = 0; i < kTurns<kDim>; ++i)
      if (first + i * kGroups < all) work(first, i);
  }
}

template <int kDim>
cudaError_t launch_append(const Append& a, bool halves, bool e4m3, cudaStream_t stream) {
  auto kernel = halves ? (e4m3 ? append_paged_k<kDim, true, true> : append_paged_k<kDim, true, false>)
                       : (e4m3 ? append_paged_k<kDim, false, true> : append_paged_k<kDim, false, false>);
  return launch(kernel, dim3(static_cast<unsigned>(a.tokens)), dim3(kThreads), 0, stream, a);
}

}  // namespace
}  // namespace sl

extern "C" int sl_append_paged(const uint16_t* qkv, int64_t tokens, int heads, int kv_heads, int head_dim,
                               const float* norm_q, const float* norm_k, float eps, const float* freqs, int max_pos,
                               int pairs, const int32_t* seq, const int32_t* positions, const int32_t* table, int seqs,
                               int table_width, int64_t pages, int page_size, int cache_type, void* k_cache,
                               void* v_cache, float* k_scale, float* v_scale, uint16_t* q, void* stream) {
  using namespace sl;
  if (tokens < 0 || tokens > 0x7FFFFFFF || heads < 1 || kv_heads < 1 || heads > 65536 || kv_heads > 65536 ||
      (head_dim != 64 && head_dim != 128) || max_pos < 1 ||
      (pairs != SL_PAIRS_ADJACENT && pairs != SL_PAIRS_HALVES) || seqs < 0 || (seqs == 0 && tokens != 0) || table_width < 1 || pages < 1 ||
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

extern "C" int sl_append_paged_with(const sl_append_paged_args* a) {
  if (a == nullptr) return SL_INVALID_ARG;
  return sl_append_paged(a->qkv, a->tokens, a->heads, a->kv_heads, a->head_dim, a->norm_q, a->norm_k, a->eps, a->freqs, a->max_pos,
                         a->pairs, a->seq, a->positions, a->table, a->seqs, a->table_width, a->pages, a->page_size, a->cache_type,
                         a->k_cache, a->v_cache, a->k_scale, a->v_scale, a->q, a->stream);
}
