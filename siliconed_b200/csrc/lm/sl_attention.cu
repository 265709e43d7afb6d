// The attention of one new token per sequence over the paged key-value cache (sl_paged_attention).
//
//   s_t = scale q . k_t,  p_t = exp(s_t - m),  out = sum p_t v_t / sum p_t,  lse = m + log(sum p_t)
//
// One pass over the cache with a running maximum and sum (the online softmax).  Bound by HBM: every key and value of
// the contexts is read once and used for the heads / kv_heads query heads that share it, 2 to 4 operations a byte
// and query head.
//
// Work.  The contexts of all (sequence, key-value head) pairs are laid end to end in units of 64 tokens, and every
// CTA takes an equal share of consecutive units, whatever the lengths are: a share may end one pair's context and
// begin the next one's.  A context that lies in one share is finished there.  Where a context is cut between
// CTAs each writes its part's maximum, sum and unnormalised output to the workspace; the last to arrive (a counter
// that it sets back to zero) adds the parts in the order of the shares, so every call gives the same bits.  A CTA
// leaves at most two parts (its first and its last context), so the workspace does not grow with the batch.
//
// Inside a CTA each of the 4 warps takes tiles of 16 tokens with a maximum, sum and output of its own, joined through
// shared memory at the context's end.  Both products run on mma.sync m16n8k16 with the cache as the A operand:
// S^T = K q^T (16 tokens x 8 query heads) and O^T += V^T P^T (16 dims x 8 query heads).  The reduction index of either
// product may be permuted freely when both operands agree, so every lane loads 16 consecutive bytes of a cache
// row straight into the registers that the MMA reads: nothing of the cache goes through shared memory.  At one
// query row a tcgen05 tile (128 rows) would be 94 to 99 % padding and its operands would have to be staged, rotated
// and awaited; the MMA work here is a few percent of the tensor pipe.
#include <cmath>

#include "sl_common.cuh"

namespace sl {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kTile = 16;                 // tokens of a warp's step
constexpr int kUnit = kWarps * kTile;     // tokens of a unit of work
constexpr int kCtasPerSm = 2;
constexpr int kMaxBatch = 1024;           // sequences of a launch

struct Attention {
  const uint16_t* q;
  const void *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int32_t *table, *lengths;
  int batch, heads, kv_heads, group, subs;  // subs: tiles of query heads of a key-value head
  int table_width;
  int64_t pages;
  int page_size, page_shift;                // page_shift: -1 unless the size is a power of two
  float scale_log2;                         // scale * log2(e)
  uint16_t* out;
  float* lse;
  uint32_t* counters;                       // [gridDim.x]
  float* parts;                             // [2 * gridDim.x][rows * (dim + 2)]
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An 8 x 8 tile of 16-bit values transposed across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Four e4m3 codes to bf16, exactly: the seven low bits of a code moved under bf16's exponent read as
// value * 2^-120 (subnormal codes included), so one multiplication by 2^120 finishes it.  The cache holds no NaN
// codes that matter: a NaN value makes its head's scale NaN.
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const __nv_bfloat162 up = __nv_bfloat162(__ushort_as_bfloat16(0x7B80), __ushort_as_bfloat16(0x7B80));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t p = __byte_perm(w, 0, i == 0 ? 0x1404 : 0x3424);  // code 2i in byte 1, code 2i + 1 in byte 3
    const uint32_t r = ((p & 0x7F007F00u) >> 4) | (p & 0x80008000u);
    const __nv_bfloat162 h = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&r), up);
    (i == 0 ? lo : hi) = *reinterpret_cast<const uint32_t*>(&h);
  }
}

// The share of work: CTA w of W takes units [w T / W, (w + 1) T / W); unit u belongs to CTA ((u + 1) W - 1) / T.
__device__ __forceinline__ int64_t share_start(int64_t w, int64_t total, int64_t workers) { return w * total / workers; }
__device__ __forceinline__ int64_t share_of(int64_t u, int64_t total, int64_t workers) {
  return ((u + 1) * workers - 1) / total;
}

// kNH: tiles of 8 query heads (1 or 2).
template <int kDim, bool kE4m3, int kNH>
__global__ void __launch_bounds__(kThreads, 2) paged_attention_k(const Attention a) {
  constexpr int kRows = 8 * kNH;
  constexpr int kBytes = kE4m3 ? 1 : 2;
  constexpr int kRowBytes = kDim * kBytes;
  constexpr int kKLoads = kRowBytes / 64;                 // 16-byte loads of a key row a lane: 4 lanes share a row
  constexpr int kVWidth = kRowBytes >= 128 ? 16 : 8;      // bytes a lane loads of a value row: 8 lanes share a row
  constexpr int kVLoads = kRowBytes / (8 * kVWidth);
  constexpr int kVDims = kVWidth / kBytes;                // dims a lane holds of one load
  constexpr int kPairs = kDim / 16;                       // M tiles of O^T
  constexpr int kPartFloats = kRows * (kDim + 2);

  __shared__ int64_t first_unit[kMaxBatch + 1];
  __shared__ int64_t scan[kWarps];
  __shared__ float part_m[kWarps][kRows], part_l[kWarps][kRows];
  __shared__ __align__(16) float part_o[kWarps][kRows][kDim + 4];  // read 16 bytes at a time
  __shared__ int last_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  sc::pdl_launch_dependents();
  sc::pdl_wait();

  // Units of every sequence, summed: each thread takes a run of sequences.
  const int hh = a.kv_heads * a.subs;
  const int64_t room = static_cast<int64_t>(a.table_width) * a.page_size;
  {
    const int per = (a.batch + kThreads - 1) / kThreads;
    const int b0 = tid * per, b1 = min(a.batch, b0 + per);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) {
      int64_t len = a.lengths[b];
      if (len < 0 || len > room) {
        sc::record_error(a.err, kErrRange, kSiteAttentionLength);
        len = len < 0 ? 0 : room;
      }
      first_unit[b] = mine;
      mine += (len + kUnit - 1) / kUnit * hh;
    }
    int64_t sum = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t v = __shfl_up_sync(0xFFFFFFFFu, sum, off);
      if (lane >= off) sum += v;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    int64_t before = sum - mine;
    for (int w = 0; w < warp; ++w) before += scan[w];
    for (int b = b0; b < b1; ++b) first_unit[b] += before;
    if (tid == kThreads - 1) first_unit[a.batch] = before + mine;
    __syncthreads();
  }
  const int64_t total = first_unit[a.batch];

  // Sequences without tokens.
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
    if (first_unit[b + 1] == first_unit[b]) {
      uint32_t* o = reinterpret_cast<uint32_t*>(a.out + static_cast<int64_t>(b) * a.heads * kDim);
      for (int i = tid; i < a.heads * kDim / 2; i += kThreads) o[i] = 0u;
      if (a.lse != nullptr)
        for (int i = tid; i < a.heads; i += kThreads) a.lse[static_cast<int64_t>(b) * a.heads + i] = -INFINITY;
    }

  const int64_t workers = min(static_cast<int64_t>(gridDim.x), total);
  if (blockIdx.x >= workers) return;
  const int64_t u_begin = share_start(blockIdx.x, total, workers), u_end = share_start(blockIdx.x + 1, total, workers);

  for (int64_t u = u_begin; u < u_end;) {
    // The sequence, key-value head and tile of query heads of unit u: the last sequence that starts at or before it
    // (sequences without tokens share their start with the next one).
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_unit[mid] <= u) lo = mid; else hi = mid;
    }
    const int b = lo;
    const int64_t units = (first_unit[b + 1] - first_unit[b]) / hh;
    const int64_t which = (u - first_unit[b]) / units;
    const int64_t s0 = first_unit[b] + which * units, s1 = s0 + units;
    const int kvh = static_cast<int>(which) / a.subs, sub = static_cast<int>(which) % a.subs;
    const int head0 = kvh * a.group + sub * kRows;             // first query head of the tile
    const int rows = min(kRows, a.group - sub * kRows);        // query heads of the tile
    const int64_t stop = min(u_end, s1);
    const int len = static_cast<int>(min(max(static_cast<int64_t>(a.lengths[b]), int64_t(0)), room));
    const int t_begin = static_cast<int>((u - s0) * kUnit);
    const int t_end = static_cast<int>(min(static_cast<int64_t>(len), (stop - s0) * kUnit));
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.table_width;

    // q as the B operand of S^T: query head g of each tile of 8, the dims in the order of the key loads.
    uint32_t qf[kNH][kDim / 8];
#pragma unroll
    for (int n = 0; n < kNH; ++n) {
      const bool there = n * 8 + g < rows;
      const uint4* src = reinterpret_cast<const uint4*>(a.q + (static_cast<int64_t>(b) * a.heads + head0 + n * 8 + g) * kDim);
#pragma unroll
      for (int j = 0; j < kDim / 32; ++j) {
        // bf16 cache: load j of a key row holds dims 32 j + 8 c ..; e4m3: dims 64 j + 16 c ..
        const int at = kE4m3 ? (j >> 1) * 8 + c * 2 + (j & 1) : j * 4 + c;
        const uint4 v = there ? src[at] : make_uint4(0, 0, 0, 0);
        qf[n][4 * j] = v.x, qf[n][4 * j + 1] = v.y, qf[n][4 * j + 2] = v.z, qf[n][4 * j + 3] = v.w;
      }
    }
    float m[kNH][2], l[kNH][2];  // of query heads 2 c and 2 c + 1 of each tile; l is this lane's own sum
    float o[kNH][kPairs][4];
#pragma unroll
    for (int n = 0; n < kNH; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
    }

    for (int t0 = t_begin + warp * kTile; t0 < t_end; t0 += kUnit) {
      // The cache row of token t0 + (lane & 15), all ones where there is none.
      uint32_t row = 0xFFFFFFFFu;
      {
        const int t = t0 + (lane & 15);
        if (t < t_end) {
          const int index = a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size;
          const int page = table[index];
          if (page < 0 || page >= a.pages)
            sc::record_error(a.err, kErrRange, kSiteAttentionPage);
          else
            row = (static_cast<uint32_t>(page) * a.kv_heads + kvh) * a.page_size + (t - index * a.page_size);
        }
      }
      uint32_t kr[2], vr[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) kr[i] = __shfl_sync(0xFFFFFFFFu, row, g + 8 * i);
#pragma unroll
      for (int i = 0; i < 4; ++i) vr[i] = __shfl_sync(0xFFFFFFFFu, row, 2 * c + (i & 1) + 8 * (i >> 1));
      uint4 kd[2][kKLoads];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(a.k_cache) +
                                                          static_cast<uint64_t>(kr[i]) * kRowBytes) + c;
#pragma unroll
        for (int j = 0; j < kKLoads; ++j)
          kd[i][j] = kr[i] != 0xFFFFFFFFu ? __ldcs(src + 4 * j) : make_uint4(0, 0, 0, 0);
      }
      uint32_t vd[4][kVLoads][kVWidth / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* src = static_cast<const char*>(a.v_cache) + static_cast<uint64_t>(vr[i]) * kRowBytes + g * kVWidth;
#pragma unroll
        for (int e = 0; e < kVLoads; ++e) {
          if (kVWidth == 16) {
            const uint4 v = vr[i] != 0xFFFFFFFFu ? __ldcs(reinterpret_cast<const uint4*>(src + e * 128)) : make_uint4(0, 0, 0, 0);
            vd[i][e][0] = v.x, vd[i][e][1] = v.y, vd[i][e][kVWidth / 4 - 2] = v.z, vd[i][e][kVWidth / 4 - 1] = v.w;
          } else {
            const uint2 v = vr[i] != 0xFFFFFFFFu ? __ldcs(reinterpret_cast<const uint2*>(src + e * 64)) : make_uint2(0, 0);
            vd[i][e][0] = v.x, vd[i][e][1] = v.y;
          }
        }
      }
      float ks[2] = {1.0f, 1.0f}, vs[2] = {1.0f, 1.0f};  // of tokens g and g + 8
      if (kE4m3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ks[i] = kr[i] != 0xFFFFFFFFu ? a.k_scale[kr[i]] : 0.0f;
          vs[i] = kr[i] != 0xFFFFFFFFu ? a.v_scale[kr[i]] : 0.0f;
        }
      }

      // S^T: tokens g and g + 8 by query heads 2 c and 2 c + 1.
      float s[kNH][4];
#pragma unroll
      for (int n = 0; n < kNH; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < kKLoads; ++j) {
        const uint32_t w0[4] = {kd[0][j].x, kd[0][j].y, kd[0][j].z, kd[0][j].w};
        const uint32_t w1[4] = {kd[1][j].x, kd[1][j].y, kd[1][j].z, kd[1][j].w};
        if (kE4m3) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_bf16(w0[i], a0, a2);
            e4m3x4_to_bf16(w1[i], a1, a3);
#pragma unroll
            for (int n = 0; n < kNH; ++n) mma16816(s[n], a0, a1, a2, a3, qf[n][8 * j + 2 * i], qf[n][8 * j + 2 * i + 1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < kNH; ++n)
              mma16816(s[n], w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1], qf[n][4 * j + 2 * i],
                       qf[n][4 * j + 2 * i + 1]);
        }
      }
      uint32_t p[kNH][2];  // P^T as the B operand: head g, tokens 2 c, 2 c + 1 and 2 c + 8, 2 c + 9
      const bool there0 = kr[0] != 0xFFFFFFFFu, there1 = kr[1] != 0xFFFFFFFFu;
#pragma unroll
      for (int n = 0; n < kNH; ++n) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = (i < 2 ? there0 : there1) ? s[n][i] * (kE4m3 ? ks[i >> 1] * a.scale_log2 : a.scale_log2) : -INFINITY;
        float top[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], off));
          top[1] = fmaxf(top[1], __shfl_xor_sync(0xFFFFFFFFu, top[1], off));
        }
        float base[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float now = fmaxf(m[n][i], top[i]);
          base[i] = now == -INFINITY ? 0.0f : now;  // nothing but -inf so far: every p is 0
          top[i] = ex2(m[n][i] - base[i]);          // the factor of what was summed before
          m[n][i] = now;
        }
        if (__any_sync(0xFFFFFFFFu, top[0] != 1.0f || top[1] != 1.0f)) {
          l[n][0] *= top[0];
          l[n][1] *= top[1];
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            o[n][i][0] *= top[0];
            o[n][i][1] *= top[1];
            o[n][i][2] *= top[0];
            o[n][i][3] *= top[1];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ex2(x[i] - base[i & 1]);
        l[n][0] += x[0] + x[2];
        l[n][1] += x[1] + x[3];
        // The one rounding to 16 bits: p (times its token's scale of v) as the MMA's operand.
        p[n][0] = transpose8x8(pack_bf16x2(x[0] * vs[0], x[1] * vs[0]));
        p[n][1] = transpose8x8(pack_bf16x2(x[2] * vs[1], x[3] * vs[1]));
      }
      // O^T += V^T P^T.  M tile i of load e: rows g are dims (8 e + g) kVDims + 2 i, rows g + 8 the dims after them.
#pragma unroll
      for (int e = 0; e < kVLoads; ++e)
#pragma unroll
        for (int w = 0; w < kVWidth / 4; ++w) {
          if (kE4m3) {
            uint32_t lo4[4], hi4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e4m3x4_to_bf16(vd[i][e][w], lo4[i], hi4[i]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t* r = half == 0 ? lo4 : hi4;
              const uint32_t a0 = __byte_perm(r[0], r[1], 0x5410), a1 = __byte_perm(r[0], r[1], 0x7632);
              const uint32_t a2 = __byte_perm(r[2], r[3], 0x5410), a3 = __byte_perm(r[2], r[3], 0x7632);
#pragma unroll
              for (int n = 0; n < kNH; ++n)
                mma16816(o[n][e * (kVDims / 2) + 2 * w + half], a0, a1, a2, a3, p[n][0], p[n][1]);
            }
          } else {
            const uint32_t a0 = __byte_perm(vd[0][e][w], vd[1][e][w], 0x5410), a1 = __byte_perm(vd[0][e][w], vd[1][e][w], 0x7632);
            const uint32_t a2 = __byte_perm(vd[2][e][w], vd[3][e][w], 0x5410), a3 = __byte_perm(vd[2][e][w], vd[3][e][w], 0x7632);
#pragma unroll
            for (int n = 0; n < kNH; ++n) mma16816(o[n][e * (kVDims / 2) + w], a0, a1, a2, a3, p[n][0], p[n][1]);
          }
        }
    }

    // Join the warps.
    __syncthreads();  // the arrays are free (an earlier context's readers are done)
#pragma unroll
    for (int n = 0; n < kNH; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][i] += __shfl_xor_sync(0xFFFFFFFFu, l[n][i], off);
        if (g == 0) {
          part_m[warp][n * 8 + 2 * c + i] = m[n][i];
          part_l[warp][n * 8 + 2 * c + i] = l[n][i];
        }
#pragma unroll
        for (int e = 0; e < kVLoads; ++e)
#pragma unroll
          for (int w = 0; w < kVDims / 2; ++w) {
            const float* acc = o[n][e * (kVDims / 2) + w];
            float* dst = &part_o[warp][n * 8 + 2 * c + i][(8 * e + g) * kVDims + 2 * w];
            *reinterpret_cast<float2*>(dst) = make_float2(acc[i], acc[2 + i]);
          }
      }
    __syncthreads();
    const bool whole = u == s0 && stop == s1;
    // Every thread: a run of 4 dims of the rows r0, r0 + step, ...
    constexpr int kRun = kDim / 4, kStep = kThreads / kRun > 0 ? kThreads / kRun : 1;
    const int slot = u == u_begin ? 0 : 1;
    float* part = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * kPartFloats;
    for (int r = tid / kRun; r < rows; r += kStep) {
      const int d0 = (tid % kRun) * 4;
      float top = part_m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, part_m[w][r]);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(part_m[w][r] - base);
        const float4 v = *reinterpret_cast<const float4*>(&part_o[w][r][d0]);
        sum += f * part_l[w][r];
        acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
      }
      if (whole) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t head = static_cast<int64_t>(b) * a.heads + head0 + r;
        *reinterpret_cast<uint2*>(a.out + head * kDim + d0) =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        if (d0 == 0 && a.lse != nullptr) a.lse[head] = sum == 0.0f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float4*>(part + r * kDim + d0) = acc;
        if (d0 == 0) *reinterpret_cast<float2*>(part + kRows * kDim + 2 * r) = make_float2(top, sum);
      }
    }
    if (!whole) {
      // The last of the context's CTAs adds the parts, in the order of the shares.
      const int64_t wa = share_of(s0, total, workers), wb = share_of(s1 - 1, total, workers);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const uint32_t before = atomicAdd(a.counters + wa, 1u);
        last_flag = before == static_cast<uint32_t>(wb - wa);
        if (last_flag) a.counters[wa] = 0u;
        __threadfence();
      }
      __syncthreads();
      if (last_flag) {
        for (int r = tid / kRun; r < rows; r += kStep) {
          const int d0 = (tid % kRun) * 4;
          float top = -INFINITY, sum = 0.0f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int64_t w = wa; w <= wb; ++w) {
            const float* src = a.parts + (w * 2 + (share_start(w, total, workers) < s0 ? 1 : 0)) * kPartFloats;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + kRows * kDim + 2 * r));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(src + r * kDim + d0));
            const float now = fmaxf(top, ml.x), base = now == -INFINITY ? 0.0f : now;
            const float f0 = ex2(top - base), f1 = ex2(ml.x - base);
            sum = sum * f0 + ml.y * f1;
            acc.x = acc.x * f0 + v.x * f1, acc.y = acc.y * f0 + v.y * f1;
            acc.z = acc.z * f0 + v.z * f1, acc.w = acc.w * f0 + v.w * f1;
            top = now;
          }
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          const int64_t head = static_cast<int64_t>(b) * a.heads + head0 + r;
          *reinterpret_cast<uint2*>(a.out + head * kDim + d0) =
              make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
          if (d0 == 0 && a.lse != nullptr) a.lse[head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        }
      }
    }
    u = stop;
  }
}

template <int kDim, bool kE4m3, int kNH>
cudaError_t launch_attention(const Attention& a, int workers, cudaStream_t stream) {
  return launch(paged_attention_k<kDim, kE4m3, kNH>, dim3(static_cast<unsigned>(workers)), dim3(kThreads), 0, stream, a);
}

template <int kDim>
cudaError_t launch_dim(const Attention& a, bool e4m3, int workers, cudaStream_t stream) {
  if (a.group <= 8)
    return e4m3 ? launch_attention<kDim, true, 1>(a, workers, stream) : launch_attention<kDim, false, 1>(a, workers, stream);
  return e4m3 ? launch_attention<kDim, true, 2>(a, workers, stream) : launch_attention<kDim, false, 2>(a, workers, stream);
}

// The SMs of the current device (0: none).
int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return n;
}

bool shape_ok(int heads, int kv_heads, int head_dim) {
  return heads >= 1 && kv_heads >= 1 && heads <= 65536 && heads % kv_heads == 0 &&
         (head_dim == 64 || head_dim == 128);
}

int tile_rows(int heads, int kv_heads) { return heads / kv_heads <= 8 ? 8 : 16; }

// Counters, rounded up to 16 bytes, then two parts a worker.
size_t counter_bytes(int workers) { return (static_cast<size_t>(workers) * 4 + 15) / 16 * 16; }

}  // namespace
}  // namespace sl

extern "C" int sl_paged_attention_workspace(int heads, int kv_heads, int head_dim, size_t* bytes) {
  using namespace sl;
  if (bytes == nullptr || !shape_ok(heads, kv_heads, head_dim)) return SL_INVALID_ARG;
  const int sms = sm_count();
  if (sms == 0) return SL_CUDA_ERROR;
  const int workers = sms * kCtasPerSm;
  *bytes = counter_bytes(workers) +
           static_cast<size_t>(workers) * 2 * tile_rows(heads, kv_heads) * (head_dim + 2) * sizeof(float);
  return SL_OK;
}

extern "C" int sl_paged_attention(const uint16_t* q, const void* k_cache, const void* v_cache, const float* k_scale,
                                  const float* v_scale, int cache_type, const int32_t* table, const int32_t* lengths,
                                  int batch, int heads, int kv_heads, int head_dim, int table_width, int64_t pages,
                                  int page_size, float scale, uint16_t* out, float* lse, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace sl;
  if (batch < 0 || !shape_ok(heads, kv_heads, head_dim) || table_width < 1 || pages < 1 || page_size < 1 ||
      (cache_type != SL_BF16 && cache_type != SL_E4M3) || !std::isfinite(scale))
    return SL_INVALID_ARG;
  // Cache rows and a sequence's tokens are counted in 32 bits.
  if (pages > 0x7FFFFFFF || static_cast<double>(pages) * kv_heads * page_size >= 4294967295.0 ||
      static_cast<int64_t>(table_width) * page_size > 0x7FFFFFC0)
    return SL_INVALID_ARG;
  if (batch == 0) return SL_OK;
  for (const void* p : {static_cast<const void*>(q), k_cache, v_cache, static_cast<const void*>(out),
                        static_cast<const void*>(workspace)})
    if (p == nullptr || !aligned(p, 16)) return SL_INVALID_ARG;
  if (table == nullptr || lengths == nullptr || !aligned(table, 4) || !aligned(lengths, 4) || !aligned(lse, 4))
    return SL_INVALID_ARG;
  const bool e4m3 = cache_type == SL_E4M3;
  if (e4m3 != (k_scale != nullptr) || e4m3 != (v_scale != nullptr) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return SL_INVALID_ARG;
  size_t need = 0;
  if (const int s = sl_paged_attention_workspace(heads, kv_heads, head_dim, &need); s != SL_OK) return s;
  if (workspace_bytes < need) return SL_INVALID_ARG;
  const int workers = sm_count() * kCtasPerSm;
  int* err = error_word();
  if (err == nullptr) return SL_CUDA_ERROR;
  const int group = heads / kv_heads;
  int shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    for (shift = 0; (1 << shift) < page_size;) ++shift;
  const float scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  for (int b0 = 0; b0 < batch; b0 += kMaxBatch) {
    const int64_t at = static_cast<int64_t>(b0) * heads;
    const Attention a{q + at * head_dim,
                      k_cache,
                      v_cache,
                      k_scale,
                      v_scale,
                      table + static_cast<int64_t>(b0) * table_width,
                      lengths + b0,
                      batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch,
                      heads,
                      kv_heads,
                      group,
                      (group + tile_rows(heads, kv_heads) - 1) / tile_rows(heads, kv_heads),
                      table_width,
                      pages,
                      page_size,
                      shift,
                      scale_log2,
                      out + at * head_dim,
                      lse == nullptr ? nullptr : lse + at,
                      static_cast<uint32_t*>(workspace),
                      reinterpret_cast<float*>(static_cast<char*>(workspace) + counter_bytes(workers)),
                      err};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = head_dim == 64 ? launch_dim<64>(a, e4m3, workers, st)
                                         : launch_dim<128>(a, e4m3, workers, st);
    if (e != cudaSuccess) return status_of(e);
  }
  return SL_OK;
}
