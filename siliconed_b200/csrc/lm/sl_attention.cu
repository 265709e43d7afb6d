// The attention of one new token per sequence over the paged key-value cache (sl_paged_attention).
//
//   s_t = scale q . k_t,  p_t = exp(s_t - m),  out = sum p_t v_t / sum p_t,  lse = m + log(sum p_t)
//
// One pass over the cache with a running maximum and sum (the online softmax).  Bound by HBM: every key and value of
// the contexts is read once and used for the heads / kv_heads query heads that share it, 2 to 4 operations a byte
// and query head.  Measured (B200, 32 query on 8 key-value heads of 128, calls after one another): 8 contexts of 65536 tokens
// in bf16 6.4 TB/s (0.99 of a copy's rate), in e4m3 6.2; 33 ragged contexts of up to 4400 tokens 5.4; one context of
// 131072 (4 key-value heads) 54 us, 5.0 TB/s, of 513 tokens 9 us, of 16 tokens 5 us.
//
// Work.  The contexts of all (sequence, key-value head) pairs are laid end to end in units (a step of every warp of a
// CTA, plus one per context) and every CTA takes an equal share of consecutive units, whatever the lengths are: a share
// may end one pair's context and begin the next one's.  A context that lies in one share is finished there.  Where a
// context is cut between CTAs each writes its part's maximum, sum and unnormalised output to the workspace; the last to
// arrive (a counter that it sets back to zero) adds the parts in the order of the shares, so every call gives the same
// bits.  A CTA leaves at most two parts (its first and its last context), so the workspace does not grow with the batch.
// (A queue that hands out the last quarter of the units in smaller pieces measured no faster.  The share worked out and its
// first unit brought to L2 while the kernel before this one ends: 2 % faster in a chain of long calls, 2 us slower alone.)
//
// Inside a CTA each warp takes steps of 32 tokens with a maximum, sum and output of its own, joined through shared
// memory at the context's end.  Both products run on mma.sync m16n8k16 with the cache as the A operand:
// S^T = K q^T (16 tokens x 8 query heads) and O^T += V^T P^T (16 dims x 8 query heads).  The reduction index of either
// product may be permuted freely when both operands agree, so every lane reads 16 consecutive bytes of a cache row as
// the registers of its MMA fragments: no transposition, no ldmatrix.  At one query row a tcgen05 tile (128 rows) would
// be 94 to 99 % padding and its operands would have to be rearranged and awaited; the MMA work here is a few percent
// of the tensor pipe.
//
// The cache reaches shared memory by bulk copies (cp.async.bulk) that each warp issues for itself, two to three steps
// ahead: token rows that follow one another in a page are one copy, whatever the page size; every lane looks up one
// token.  (Measured on the way: 16-byte cp.async by every lane read 5.2 TB/s, bound by the 170 instructions a step
// of addresses and copies; a copy kernel of bulk copies alone reads 6.8 TB/s in rows of 256 bytes, 4.2 in rows of 128,
// 7.1 in runs of 16 rows.)
//
// An e4m3 cache runs in f16: codes are exact in it, q is first brought to a largest magnitude in [1, 2) by a power of
// two per head, and p times its token's scale is taken relative to the largest scale so far (a second running
// maximum), times 2^15, so that it uses f16's whole range.
#include <cuda_fp16.h>

#include <cmath>

#include "sl_common.cuh"
#include "sl_ring.cuh"

namespace sl {
namespace {

constexpr int kStep = 32;                 // tokens of a warp's step: two MMA tiles of 16
constexpr int kMaxBatch = 512;            // sequences of a launch

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

// What scores are taken relative to: their maximum, but 0 where that is -inf (every p is 0 then, not NaN) or +inf (the sum is
// +inf then, and so is its logarithm).
__device__ __forceinline__ float zero_of(float top) { return fabsf(top) == INFINITY ? 0.0f : top; }

template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (kHalf)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
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

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four e4m3 codes to f16, exactly (NaN codes to NaN): codes 0 and 1, codes 2 and 3.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// An asynchronous copy of 4 bytes to shared memory, zeros where `there` is false.
__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// The shares of `total` units among `workers` CTAs: consecutive, the first `extra` of them one unit longer.  Counted in 32
// bits (the launch sees to it): a 64-bit division takes as long as a step's products.
struct Shares {
  uint32_t workers, each, extra;
  __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * each + min(w, extra); }
  __device__ __forceinline__ uint32_t of(uint32_t u) const {
    const uint32_t longer = extra * (each + 1);
    return u < longer ? u / (each + 1) : extra + (u - longer) / each;
  }
};

// Adds one and returns the count before: what this CTA wrote before is seen by whoever counts after it.
__device__ __forceinline__ uint32_t count_arrival(uint32_t* counter) {
  uint32_t before;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

// Geometry of a step's 32 tokens in shared memory: rows in order.  Lane (g, c) reads bytes 64 j + 16 c .. of the key rows
// g + 8 i, i < 4 (two lanes a bank), and kVWidth bytes at 8 e kVWidth + g kVWidth of the value rows 16 t + 2 c, + 1, + 8,
// + 9: value rows of 256 bytes are copied one by one, 272 bytes apart, so that these reads meet no bank twice; shorter
// ones in runs, since copies of 128 bytes are too many, at four lanes a bank (half of shared memory's rate then).
// A warp's ring has kSlots slots that take a step's keys, its values, the next step's keys and so on.
// kWide: one CTA an SM, for few contexts: a long context is cut into fewer parts, and more threads add them.  Else
// CTAs of 4 warps, for many contexts: one begins while another ends.
template <int kDim, bool kE4m3, int kNH, bool kWide>
struct Shape {
  static constexpr int kRows = 8 * kNH;
  static constexpr int kRowBytes = kDim * (kE4m3 ? 1 : 2);
  static constexpr bool kBig = kRowBytes >= 256;
  // By shared memory and registers (248, 168 or 128 a thread).  Rows of 128 bytes or less are bound by the warps' latency
  // rather than by the copies ahead: 16 warps with one step's copies each read 6.2 TB/s of an e4m3 cache, 12 with two
  // steps' 5.8, 8 with three steps' 4.9.
  static constexpr int kWarpsPerSm = kBig || (kNH == 2 && kDim == 128) ? 8 : kNH == 2 ? 12 : 16;
  static constexpr int kWarps = kWide ? kWarpsPerSm : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCtasPerSm = kWarpsPerSm / kWarps;
  static constexpr int kUnit = kWarps * kStep;                  // tokens of a unit of work
  static constexpr int kKLoads = kRowBytes / 64;
  static constexpr int kVWidth = kRowBytes >= 128 ? 16 : 8;
  static constexpr int kVLoads = kRowBytes / (8 * kVWidth);
  static constexpr int kVDims = kVWidth / (kE4m3 ? 1 : 2);
  static constexpr int kVPitch = kBig ? kRowBytes + 16 : kRowBytes;
  static constexpr int kSlotBytes = kStep * kVPitch;
  static constexpr int kSlots = kBig ? 3 : (kRowBytes >= 128 ? 2 : 4) * (kWarpsPerSm == 16 ? 1 : 2);
  static constexpr int kAhead = (kSlots + 1) / 2;               // steps begun before a step is used
  static constexpr int kScaleAt = kSlots * kSlotBytes;          // e4m3: scales of kAhead + 1 steps, 32 of k and 32 of v
  static constexpr int kWarpBytes = kScaleAt + (kE4m3 ? (kAhead + 1) * 256 : 0);  // reused for the join
  static constexpr int kSmem = kWarps * kWarpBytes;
  static constexpr int kPartRow = kDim + 4;
  static constexpr int kPartFloats = kRows * (kDim + 2);
  // A launch's shared memory on `workers` CTAs.  The ring also holds the factors of a cut context's parts when they are added,
  // a float a row and part, and one context may be cut over every CTA.  (Two floats: 592 parts of 8 rows pass the four-warp
  // shapes' rings of 32 to 35 KB, and the 3 KB more take so much of the L1 that 64 ragged e4m3 contexts are 1.7 % slower.)
  static constexpr int smem_bytes(int workers) {
    const int factors = kRows * workers * static_cast<int>(sizeof(float));
    return factors > kSmem ? factors : kSmem;
  }
  static_assert(kRows * kPartRow * 4 <= kWarpBytes, "the join's part fits the ring");
  static_assert(!kE4m3 || kSlots % 2 == 0, "the scales go with whole steps");
  static_assert(smem_bytes(148 * kCtasPerSm) == kSmem, "a B200's rings hold the factors of as many parts as there are CTAs");
};
constexpr int kMostCtasPerSm = 4;

// kNH: tiles of 8 query heads (1 or 2).
template <int kDim, bool kE4m3, int kNH, bool kWide>
__global__ void __launch_bounds__(Shape<kDim, kE4m3, kNH, kWide>::kThreads, Shape<kDim, kE4m3, kNH, kWide>::kCtasPerSm)
    paged_attention_k(const Attention a) {
  using S = Shape<kDim, kE4m3, kNH, kWide>;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kUnit = S::kUnit;
  constexpr int kRows = S::kRows, kRowBytes = S::kRowBytes, kKLoads = S::kKLoads, kVWidth = S::kVWidth;
  constexpr int kVLoads = S::kVLoads, kVDims = S::kVDims, kSlots = S::kSlots, kAhead = S::kAhead, kVPitch = S::kVPitch, kPartFloats = S::kPartFloats;
  constexpr int kPairs = kDim / 16;  // M tiles of O^T

  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint32_t first_unit[kMaxBatch + 1];
  __shared__ int length[kMaxBatch];
  __shared__ uint32_t scan[kWarps];
  __shared__ float part_m[kWarps][kRows], part_l[kWarps][kRows];
  __shared__ uint64_t arrived[kWarps][kSlots];
  __shared__ int last_flag, abort_flag;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  sc::pdl_launch_dependents();
  if (tid < kWarps * kSlots) sc::mbar_init(&arrived[0][0] + tid, 1);
  if (tid == 0) abort_flag = 0;
  sc::fence_mbar_init();
  Ring<kSlots> order;  // of the warp's copies
  const uint32_t base = sc::smem_u32(ring) + warp * S::kWarpBytes;
  const uint8_t* const mine = ring + warp * S::kWarpBytes;
  sc::pdl_wait();

  // Units of every sequence, summed: each thread takes a run of sequences.
  const uint32_t hh = a.kv_heads * a.subs;
  const int room = a.table_width * a.page_size;
  {
    const int per = (a.batch + kThreads - 1) / kThreads;
    const int b0 = tid * per, b1 = min(a.batch, b0 + per);
    uint32_t own = 0;
    for (int b = b0; b < b1; ++b) {
      int len = a.lengths[b];
      if (len < 0 || len > room) {
        sc::record_error(a.err, kErrRange, kSiteAttentionLength);
        len = len < 0 ? 0 : room;
      }
      length[b] = len;
      first_unit[b] = own;
      // One unit more than the tokens fill stands for a context's beginning and end, which cost about as much (ragged
      // batches 6 to 13 % faster than with the tokens alone).  A share that holds nothing else leaves an empty part.
      own += len == 0 ? 0u : (static_cast<uint32_t>(len + kUnit - 1) / kUnit + 1) * hh;
    }
    uint32_t sum = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, sum, off);
      if (lane >= off) sum += v;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    uint32_t before = sum - own;
    for (int w = 0; w < warp; ++w) before += scan[w];
    for (int b = b0; b < b1; ++b) first_unit[b] += before;
    if (tid == kThreads - 1) first_unit[a.batch] = before + own;
    __syncthreads();
  }
  const uint32_t total = first_unit[a.batch];

  // Sequences without tokens.
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
    if (first_unit[b + 1] == first_unit[b]) {
      uint32_t* o = reinterpret_cast<uint32_t*>(a.out + static_cast<int64_t>(b) * a.heads * kDim);
      for (int i = tid; i < a.heads * kDim / 2; i += kThreads) o[i] = 0u;
      if (a.lse != nullptr)
        for (int i = tid; i < a.heads; i += kThreads) a.lse[static_cast<int64_t>(b) * a.heads + i] = -INFINITY;
    }

  Shares shares;
  shares.workers = min(gridDim.x, total);
  if (blockIdx.x >= shares.workers) return;
  shares.each = total / shares.workers;
  shares.extra = total % shares.workers;
  const uint32_t u_begin = shares.start(blockIdx.x), u_end = shares.start(blockIdx.x + 1);

  for (uint32_t u = u_begin; u < u_end;) {
    // The sequence, key-value head and tile of query heads of unit u: the last sequence that starts at or before it
    // (sequences without tokens share their start with the next one).
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_unit[mid] <= u) lo = mid; else hi = mid;
    }
    const int b = lo;
    const uint32_t units = (first_unit[b + 1] - first_unit[b]) / hh;
    const uint32_t which = (u - first_unit[b]) / units;
    const uint32_t s0 = first_unit[b] + which * units, s1 = s0 + units;
    const int kvh = static_cast<int>(which) / a.subs, sub = static_cast<int>(which) % a.subs;
    const int head0 = kvh * a.group + sub * kRows;             // first query head of the tile
    const int rows = min(kRows, a.group - sub * kRows);        // query heads of the tile
    const uint32_t stop = min(u_end, s1);
    const int t_begin = static_cast<int>(u - s0) * kUnit;
    const int t_end = min(length[b], static_cast<int>(stop - s0) * kUnit);
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.table_width;

    // q as the B operand of S^T: query head g of each tile of 8, the dims in the order of the key loads.
    uint32_t qf[kNH][kDim / 8];
    float unit[kNH][2];  // of query heads 2 c and 2 c + 1: a score's factor, log2(e) included
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
      unit[n][0] = unit[n][1] = a.scale_log2;
      if (kE4m3) {
        uint32_t top = 0;  // the exponent of the head's largest magnitude, in bf16's bits
#pragma unroll
        for (int j = 0; j < kDim / 8; ++j) top = max(top, max(qf[n][j] & 0x7F80u, (qf[n][j] >> 16) & 0x7F80u));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const int e = min(max(static_cast<int>(top >> 7), 1), 253);  // 2^(127 - e) and 2^(e - 127) are normal
        const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
        for (int j = 0; j < kDim / 8; ++j)
          qf[n][j] = pack_f16x2(__uint_as_float(qf[n][j] << 16) * down, __uint_as_float(qf[n][j] & 0xFFFF0000u) * down);
#pragma unroll
        for (int i = 0; i < 2; ++i) unit[n][i] *= __shfl_sync(0xFFFFFFFFu, up, (2 * c + i) * 4);
      }
    }
    float m[kNH][2], l[kNH][2];  // of query heads 2 c and 2 c + 1 of each tile; l is this lane's own sum
    float o[kNH][kPairs][4];
    float vtop = 0.0f;           // e4m3: the largest scale of v so far; o is in units of vtop 2^-15
#pragma unroll
    for (int n = 0; n < kNH; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
    }

    // The page of token t + lane (-1: none), asked for one step before it is used.
    auto page_of = [&](int t) -> int {
      t += lane;
      return t < t_end ? table[a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size] : -1;
    };
    // The tokens of a step, one a lane: its cache row, whether there is one (`there` is the mask of all lanes), and the
    // count of rows that follow one another in the cache from here on (0 inside such a run).
    struct Tokens {
      uint32_t row, there;
      int run;
    };
    auto tokens_of = [&](int t, int page) {
      Tokens k;
      const bool there = t + lane < t_end && page >= 0 && page < a.pages;
      if (t + lane < t_end && !there) sc::record_error(a.err, kErrRange, kSiteAttentionPage);
      k.row = (static_cast<uint32_t>(page) * a.kv_heads + kvh) * a.page_size +
              (a.page_shift >= 0 ? (t + lane) & (a.page_size - 1) : (t + lane) % a.page_size);
      k.there = __ballot_sync(0xFFFFFFFFu, there);
      const uint32_t before = __shfl_up_sync(0xFFFFFFFFu, k.row, 1);
      const bool starts = there && (lane == 0 || !((k.there >> (lane - 1)) & 1) || before + 1 != k.row);
      const uint32_t ends = (__ballot_sync(0xFFFFFFFFu, starts) | ~k.there) & (0xFFFFFFFEu << lane);
      k.run = starts ? (ends != 0 ? __ffs(ends) - 1 : 32) - lane : 0;
      return k;
    };
    // The keys (values) of a step on their way into the next slot.
    auto next_slot = [&](const Tokens& k) {
      uint64_t* bar = &arrived[warp][order.fill];
      if (lane == 0) sc::mbar_arrive_expect_tx(bar, __popc(k.there) * kRowBytes);
      __syncwarp();
      return bar;
    };
    auto copy = [&](uint32_t dst, const void* cache, uint32_t row, int count, uint64_t* bar) {
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                   "l"(static_cast<const char*>(cache) + static_cast<uint64_t>(row) * kRowBytes), "r"(count * kRowBytes),
                   "r"(sc::smem_u32(bar))
                   : "memory");
    };
    auto fetch_keys = [&](const Tokens& k) {
      uint64_t* bar = next_slot(k);
      if (k.run != 0) copy(base + order.fill * S::kSlotBytes + lane * kRowBytes, a.k_cache, k.row, k.run, bar);
      order.filled();
    };
    auto fetch_values = [&](const Tokens& k) {
      uint64_t* bar = next_slot(k);
      const uint32_t dst = base + order.fill * S::kSlotBytes + lane * kVPitch;
      if (S::kBig ? (k.there >> lane) & 1 : k.run != 0) copy(dst, a.v_cache, k.row, S::kBig ? 1 : k.run, bar);
      if (!((k.there >> lane) & 1)) {  // zeros where there is no token: p is 0 there, and 0 times anything finite is 0
        for (int i = 0; i < kRowBytes; i += 16)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(dst + i), "r"(0) : "memory");
        sc::fence_async_shared();  // before a later copy into the slot
      }
      order.filled();
    };
    // The oldest copy not yet used; null when it did not arrive in time: then it is still the oldest.
    auto arrival = [&]() -> const uint8_t* {
      if (!wait_warp(&arrived[warp][order.take], order.parity(), &abort_flag, a.err, kSiteAttentionCopy)) return nullptr;
      const uint8_t* at = mine + order.take * S::kSlotBytes;
      order.taken();
      return at;
    };

    // Copy n is the keys of step n / 2 (n even) or its values (n odd); copy n + kSlots goes out when copy n has been used.
    // With an odd count of slots a step's keys go out before the values of the step before them.  Pages are looked up
    // one step before the copies need them.
    // Once a wait of the CTA has given up its warps take no more steps: a barrier whose phase has not ended is not armed again.
    // The contexts' parts are written and counted all the same, so that the workspace is left ready.
    const bool halted = __any_sync(0xFFFFFFFFu, *static_cast<volatile int*>(&abort_flag)) != 0;
    const int t_first = halted ? t_end : t_begin + warp * kStep;
    bool gave_up = false;
    uint32_t masks[kAhead + 1];  // of the tokens that are there, this step's first
    Tokens held = {0, 0, 0};
    int page = page_of(t_first), scale_slot = 0;
    auto fetch_scales = [&](const Tokens& k) {
      if (kE4m3) {
        const bool there = (k.there >> lane) & 1;
        const uint32_t dst = base + S::kScaleAt + scale_slot * 256 + lane * 4;
        copy_async4(dst, a.k_scale + (there ? k.row : 0), there);
        copy_async4(dst + 128, a.v_scale + (there ? k.row : 0), there);
        copy_commit();
        scale_slot = scale_slot == kAhead ? 0 : scale_slot + 1;
      }
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int t = t_first + i * kUnit, next = page_of(t + kUnit);
      held = tokens_of(t, page);
      masks[i] = held.there;
      if (t < t_end) fetch_keys(held);
      if (t < t_end && 2 * i + 1 < kSlots) fetch_values(held);
      fetch_scales(held);
      page = next;
    }
#pragma unroll 1
    for (int t0 = t_first; t0 < t_end; t0 += kUnit) {
      // The tokens of the step kAhead on: looked at here, or with an odd count of slots once the values are used.
      const int t_ahead = t0 + kAhead * kUnit;
      auto look_ahead = [&]() {
        const int next = page_of(t_ahead + kUnit);
        held = tokens_of(t_ahead, page);
        masks[kAhead] = held.there;
        fetch_scales(held);
        page = next;
      };
      if (kSlots % 2 == 0) look_ahead();

      float ks[4], vs[4];  // of tokens g + 8 i
      if (kE4m3) {
        copy_wait<kAhead>();
        __syncwarp();  // the scales were copied by other lanes
        const float* sc = reinterpret_cast<const float*>(mine + S::kScaleAt + scale_slot * 256);  // the slot to be filled next
#pragma unroll
        for (int i = 0; i < 4; ++i) ks[i] = sc[g + 8 * i], vs[i] = sc[32 + g + 8 * i];
      }
      const uint8_t* const keys = arrival();
      if ((gave_up = keys == nullptr)) break;
      // S^T: tokens g + 8 i by query heads 2 c and 2 c + 1, in two MMA tiles.
      float s[kNH][2][4];
#pragma unroll
      for (int n = 0; n < kNH; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[n][t][0] = s[n][t][1] = s[n][t][2] = s[n][t][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < kKLoads; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint8_t* at = keys + (16 * t + g) * kRowBytes + j * 64 + c * 16;
          const uint4 k0 = *reinterpret_cast<const uint4*>(at);
          const uint4 k1 = *reinterpret_cast<const uint4*>(at + 8 * kRowBytes);
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
          if (kE4m3) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_f16(w0[i], a0, a2);
              e4m3x4_to_f16(w1[i], a1, a3);
#pragma unroll
              for (int n = 0; n < kNH; ++n)
                mma16816<true>(s[n][t], a0, a1, a2, a3, qf[n][8 * j + 2 * i], qf[n][8 * j + 2 * i + 1]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int n = 0; n < kNH; ++n)
                mma16816<false>(s[n][t], w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1], qf[n][4 * j + 2 * i],
                                qf[n][4 * j + 2 * i + 1]);
          }
        }
      __syncwarp();  // the keys' slot has been read
      if (kSlots % 2 == 0) {
        if (t_ahead < t_end) fetch_keys(held);
      } else {
        if (t_ahead - kUnit < t_end) fetch_values(held);
      }

      float vturn = 1.0f;  // e4m3: the factor of what o summed under a smaller vtop
      if (kE4m3) {
        float top = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
        if (top > vtop) {
          vturn = fmaxf(vtop, 7.9e-31f) / fmaxf(top, 7.9e-31f);
          vtop = top;
        }
        // a floor keeps the factor finite; scales below it (smaller than any that the append writes) stay exact enough
        const float f = 32768.0f / fmaxf(vtop, 7.9e-31f);
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[i] *= f;
      }
      // P^T as the B operand: head g, tokens 2 c, 2 c + 1 and 2 c + 8, 2 c + 9 of each tile.
      constexpr int kTerms = kE4m3 ? 1 : 2;
      constexpr float kTiny = 1.1754944e-38f;
      uint32_t p[kTerms][kNH][2][2];
#pragma unroll
      for (int n = 0; n < kNH; ++n) {
        float x[8];  // tokens g + 8 (i >> 1), query head 2 c + (i & 1)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = (masks[0] >> (g + 8 * (i >> 1))) & 1 ? s[n][i >> 2][i & 3] * (kE4m3 ? ks[i >> 1] * unit[n][i & 1] : unit[n][i & 1])
                                                      : -INFINITY;
        float top[2], zero[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) top[i] = fmaxf(fmaxf(x[i], x[2 + i]), fmaxf(x[4 + i], x[6 + i]));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], off));
          top[1] = fmaxf(top[1], __shfl_xor_sync(0xFFFFFFFFu, top[1], off));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float now = fmaxf(m[n][i], top[i]);
          zero[i] = zero_of(now);
          top[i] = ex2(m[n][i] - zero[i]);          // the factor of what was summed before
          m[n][i] = now;
        }
        if (__any_sync(0xFFFFFFFFu, top[0] != 1.0f || top[1] != 1.0f || vturn != 1.0f)) {
          l[n][0] *= top[0];
          l[n][1] *= top[1];
          top[0] *= vturn;
          top[1] *= vturn;
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            o[n][i][0] *= top[0];
            o[n][i][1] *= top[1];
            o[n][i][2] *= top[0];
            o[n][i][3] *= top[1];
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = ex2(x[i] - zero[i & 1]);
        l[n][0] += (x[0] + x[2]) + (x[4] + x[6]);
        l[n][1] += (x[1] + x[3]) + (x[5] + x[7]);
        // The one rounding to 16 bits, to be the MMA's operand, whose type is the cache's.  f16: p times its token's scale of v, 11
        // significant bits.  bf16: p in two terms, its upper 8 bits and the next 8 (in one term of 8 its error would stand
        // beside the output's own; the second one costs 33 ragged contexts 0.3 %, one long one 0.8 %, up to 5 % where 16 query heads
        // share a key-value head).  It is at least the smallest normal number where p is not 0: an infinity in v times it is that
        // infinity again, not NaN.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = x[2 * i], b = x[2 * i + 1];
          const uint32_t upper = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
          p[0][n][i >> 1][i & 1] = transpose8x8(kE4m3 ? pack_f16x2(a * vs[i], b * vs[i]) : upper);
          if (!kE4m3) {
            const float rest_a = fmaxf(a - __uint_as_float(__float_as_uint(a) & 0xFFFF0000u), fminf(a, kTiny));
            const float rest_b = fmaxf(b - __uint_as_float(__float_as_uint(b) & 0xFFFF0000u), fminf(b, kTiny));
            p[kTerms - 1][n][i >> 1][i & 1] = transpose8x8(pack_bf16x2(rest_a, rest_b));
          }
        }
      }
      const uint8_t* const values = arrival();
      if ((gave_up = values == nullptr)) break;
      // O^T += V^T P^T.  M tile i of load e: rows g are dims (8 e + g) kVDims + 2 i, rows g + 8 the dims after them.
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < kVLoads; ++e) {
          uint32_t v[4][kVWidth / 4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t* src = values + (16 * t + 2 * c + (i & 1) + 8 * (i >> 1)) * kVPitch + (8 * e + g) * kVWidth;
            if (kVWidth == 16) {
              const uint4 u = *reinterpret_cast<const uint4*>(src);
              v[i][0] = u.x, v[i][1] = u.y, v[i][kVWidth / 4 - 2] = u.z, v[i][kVWidth / 4 - 1] = u.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(src);
              v[i][0] = u.x, v[i][1] = u.y;
            }
          }
#pragma unroll
          for (int w = 0; w < kVWidth / 4; ++w) {
            if (kE4m3) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                uint32_t a0, a1, a2, a3;  // the codes of two tokens side by side, dim by dim
                e4m3x4_to_f16(__byte_perm(v[0][w], v[1][w], half == 0 ? 0x5140 : 0x7362), a0, a1);
                e4m3x4_to_f16(__byte_perm(v[2][w], v[3][w], half == 0 ? 0x5140 : 0x7362), a2, a3);
#pragma unroll
                for (int n = 0; n < kNH; ++n)
                  mma16816<true>(o[n][e * (kVDims / 2) + 2 * w + half], a0, a1, a2, a3, p[0][n][t][0], p[0][n][t][1]);
              }
            } else {
              const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5410), a1 = __byte_perm(v[0][w], v[1][w], 0x7632);
              const uint32_t a2 = __byte_perm(v[2][w], v[3][w], 0x5410), a3 = __byte_perm(v[2][w], v[3][w], 0x7632);
#pragma unroll
              for (int n = 0; n < kNH; ++n)
#pragma unroll
                for (int term = 0; term < kTerms; ++term)
                  mma16816<false>(o[n][e * (kVDims / 2) + w], a0, a1, a2, a3, p[term][n][t][0], p[term][n][t][1]);
            }
          }
        }
      __syncwarp();  // the values' slot has been read
      if (kSlots % 2 == 0) {
        if (t_ahead < t_end) fetch_values(held);
      } else {
        look_ahead();
        if (t_ahead < t_end) fetch_keys(held);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) masks[i] = masks[i + 1];
    }
    if (kE4m3) copy_wait<0>();
    if (gave_up) order.drain([&](uint32_t slot, uint32_t parity) { sc::mbar_wait_drain(&arrived[warp][slot], parity); });

    // Join the warps.  Each writes its part over its own ring, whose copies have all arrived (or were waited for twice).
    const float back = kE4m3 ? fmaxf(vtop, 7.9e-31f) * (1.0f / 32768.0f) : 1.0f;
    float* const part_o = reinterpret_cast<float*>(ring + warp * S::kWarpBytes);
    __syncwarp();
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
            *reinterpret_cast<float2*>(part_o + (n * 8 + 2 * c + i) * S::kPartRow + (8 * e + g) * kVDims + 2 * w) =
                make_float2(acc[i] * back, acc[2 + i] * back);
          }
      }
    __syncthreads();
    const bool whole = u == s0 && stop == s1;
    // Every thread: a run of 4 dims of the rows r0, r0 + step, ...
    constexpr int kRun = kDim / 4, kRowStep = kThreads / kRun;
    float* part = a.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (u == u_begin ? 0 : 1)) * kPartFloats;
    for (int r = tid / kRun; r < rows; r += kRowStep) {
      const int d0 = (tid % kRun) * 4;
      float top = part_m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, part_m[w][r]);
      const float zero = zero_of(top);
      float sum = 0.0f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(part_m[w][r] - zero);
        const float4 v = *reinterpret_cast<const float4*>(ring + w * S::kWarpBytes + (r * S::kPartRow + d0) * 4);
        sum += f * part_l[w][r];
        acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
      }
      if (whole) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t head = static_cast<int64_t>(b) * a.heads + head0 + r;
        *reinterpret_cast<uint2*>(a.out + head * kDim + d0) =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        if (d0 == 0 && a.lse != nullptr) a.lse[head] = sum == 0.0f ? -INFINITY : (zero + log2f(sum)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float4*>(part + r * kDim + d0) = acc;
        if (d0 == 0) *reinterpret_cast<float2*>(part + kRows * kDim + 2 * r) = make_float2(top, sum);
      }
    }
    if (!whole) {
      // The last of the context's CTAs adds the parts, in the order of the shares.
      const uint32_t wa = shares.of(s0), wb = shares.of(s1 - 1);
      __syncthreads();
      if (tid == 0) {
        last_flag = count_arrival(a.counters + wa) == wb - wa;  // after the barrier: the whole CTA's part
        if (last_flag) a.counters[wa] = 0u;
      }
      __syncthreads();
      if (last_flag) {
        // Part w lies in slot 0, but for the first one when that CTA began an earlier context.
        const int count = static_cast<int>(wb - wa) + 1;
        const float* first = a.parts + (static_cast<int64_t>(wa) * 2 + (shares.start(wa) < s0 ? 1 : 0)) * kPartFloats;
        const float* others = a.parts + static_cast<int64_t>(wa) * 2 * kPartFloats;
        auto part_of = [&](int w) { return w == 0 ? first : others + static_cast<int64_t>(w) * 2 * kPartFloats; };
        const int d0 = (tid % kRun) * 4;
        // The first parts' sums are on their way while every part's factor exp(m_w - m) is formed.
        constexpr int kEarly = 4;
        float4 early[kEarly];
#pragma unroll
        for (int w = 0; w < kEarly; ++w)
          if (w < count && tid / kRun < rows) early[w] = __ldcg(reinterpret_cast<const float4*>(part_of(w) + tid / kRun * kDim + d0));
        float* factor = reinterpret_cast<float*>(ring);  // [rows][count]: m, then exp(m - top); see smem_bytes()
        for (int r = warp; r < rows; r += kWarps) {
          float mine = -INFINITY, sum = 0.0f;  // of this lane's parts
          for (int w = lane; w < count; w += 32) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_of(w) + kRows * kDim + 2 * r));
            factor[r * count + w] = ml.x;
            const float now = fmaxf(mine, ml.x), from = zero_of(now);
            sum = sum * ex2(mine - from) + ml.y * ex2(ml.x - from);
            mine = now;
          }
          float top = mine;
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
          const float zero = zero_of(top);
          sum *= ex2(mine - zero);
          for (int w = lane; w < count; w += 32) factor[r * count + w] = ex2(factor[r * count + w] - zero);
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
          if (lane == 0) {
            part_l[0][r] = sum;
            part_m[0][r] = zero;
          }
        }
        __syncthreads();
        for (int r = tid / kRun; r < rows; r += kRowStep) {
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          const auto add = [&](float4 v, int w) {
            const float f = factor[r * count + w];
            acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
          };
          if (r == tid / kRun) {
#pragma unroll
            for (int w = 0; w < kEarly; ++w)
              if (w < count) add(early[w], w);
          } else {
            for (int w = 0; w < min(kEarly, count); ++w) add(__ldcg(reinterpret_cast<const float4*>(part_of(w) + r * kDim + d0)), w);
          }
#pragma unroll 16
          for (int w = kEarly; w < count; ++w)
            add(__ldcg(reinterpret_cast<const float4*>(others + static_cast<int64_t>(w) * 2 * kPartFloats + r * kDim + d0)), w);
          const float sum = part_l[0][r], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          const int64_t head = static_cast<int64_t>(b) * a.heads + head0 + r;
          *reinterpret_cast<uint2*>(a.out + head * kDim + d0) =
              make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
          if (d0 == 0 && a.lse != nullptr)
            a.lse[head] = sum == 0.0f ? -INFINITY : (part_m[0][r] + log2f(sum)) * 0.6931471805599453f;
        }
      }
    }
    sc::fence_async_shared();
    __syncthreads();  // the parts are read before the next context's tiles arrive
    u = stop;
  }
}

template <int kDim, bool kE4m3, int kNH, bool kWide>
cudaError_t launch_attention(const Attention& a, int sms, cudaStream_t stream) {
  using S = Shape<kDim, kE4m3, kNH, kWide>;
  auto kernel = paged_attention_k<kDim, kE4m3, kNH, kWide>;
  const int workers = sms * S::kCtasPerSm, smem = S::smem_bytes(workers);
  static unsigned long long configured = 0;  // a device's bytes are always the same; more than it has are refused
  if (const cudaError_t e = set_smem_once(kernel, smem, configured); e != cudaSuccess) return e;
  return launch(kernel, dim3(static_cast<unsigned>(workers)), dim3(S::kThreads), static_cast<size_t>(smem), stream, a);
}

template <int kDim, bool kE4m3>
cudaError_t launch_kind(const Attention& a, int sms, cudaStream_t stream) {
  // By the table's room, since the host does not know the lengths: few short contexts in a table for long ones take the wide
  // form.  Four-warp CTAs cut a long context into so many parts (444 over few contexts) that adding them costs more than the
  // switches between contexts that they hide: 4 contexts of 131072 tokens 87 us, wide 68; but 8 of 16 tokens 4.9, wide
  // 7.7, and 2048 of 128 tokens 42 either way (B200, heads of 128).
  const bool wide = static_cast<int64_t>(a.batch) * a.kv_heads * a.subs < 64 &&
                    static_cast<int64_t>(a.table_width) * a.page_size > 2048;
  if (a.group <= 8)
    return wide ? launch_attention<kDim, kE4m3, 1, true>(a, sms, stream) : launch_attention<kDim, kE4m3, 1, false>(a, sms, stream);
  return wide ? launch_attention<kDim, kE4m3, 2, true>(a, sms, stream) : launch_attention<kDim, kE4m3, 2, false>(a, sms, stream);
}

template <int kDim>
cudaError_t launch_dim(const Attention& a, bool e4m3, int sms, cudaStream_t stream) {
  return e4m3 ? launch_kind<kDim, true>(a, sms, stream) : launch_kind<kDim, false>(a, sms, stream);
}

bool shape_ok(int heads, int kv_heads, int head_dim) {
  return heads >= 1 && kv_heads >= 1 && heads <= 65536 && heads % kv_heads == 0 &&
         (head_dim == 64 || head_dim == 128);
}

int tile_rows(int heads, int kv_heads) { return heads / kv_heads <= 8 ? 8 : 16; }

// Counters, rounded up to 16 bytes, then two parts a worker.
size_t counter_bytes(int workers) { return (static_cast<size_t>(workers) * 4 + 15) / 16 * 16; }

size_t workspace_bytes_of(int sms, int heads, int kv_heads, int head_dim) {
  const int workers = sms * kMostCtasPerSm;
  return counter_bytes(workers) + static_cast<size_t>(workers) * 2 * tile_rows(heads, kv_heads) * (head_dim + 2) * sizeof(float);
}

}  // namespace
}  // namespace sl

extern "C" int sl_paged_attention_workspace(int heads, int kv_heads, int head_dim, size_t* bytes) {
  using namespace sl;
  if (bytes == nullptr || !shape_ok(heads, kv_heads, head_dim)) return SL_INVALID_ARG;
  const int sms = current_device().sms;
  if (sms == 0) return SL_CUDA_ERROR;
  *bytes = workspace_bytes_of(sms, heads, kv_heads, head_dim);
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
      static_cast<int64_t>(table_width) * page_size > 0x7FFF0000)
    return SL_INVALID_ARG;
  // So are a launch's units of 128 tokens or more.
  const int64_t most = 0x7FFFFFFFll / (((static_cast<int64_t>(table_width) * page_size + 127) / 128 + 1) * heads);
  if (most < 1) return SL_INVALID_ARG;
  const int per_launch = static_cast<int>(most < kMaxBatch ? most : kMaxBatch);
  if (batch == 0) return SL_OK;
  for (const void* p : {static_cast<const void*>(q), k_cache, v_cache, static_cast<const void*>(out),
                        static_cast<const void*>(workspace)})
    if (p == nullptr || !aligned(p, 16)) return SL_INVALID_ARG;
  if (table == nullptr || lengths == nullptr || !aligned(table, 4) || !aligned(lengths, 4) || !aligned(lse, 4))
    return SL_INVALID_ARG;
  const bool e4m3 = cache_type == SL_E4M3;
  if (e4m3 != (k_scale != nullptr) || e4m3 != (v_scale != nullptr) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return SL_INVALID_ARG;
  const Device device = current_device();
  if (device.err == nullptr) return SL_CUDA_ERROR;
  const int sms = device.sms, workers = sms * kMostCtasPerSm;
  int* const err = device.err;
  if (workspace_bytes < workspace_bytes_of(sms, heads, kv_heads, head_dim)) return SL_INVALID_ARG;
  const int group = heads / kv_heads;
  int shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    for (shift = 0; (1 << shift) < page_size;) ++shift;
  const float scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  for (int b0 = 0; b0 < batch; b0 += per_launch) {
    const int64_t at = static_cast<int64_t>(b0) * heads;
    const Attention a{q + at * head_dim,
                      k_cache,
                      v_cache,
                      k_scale,
                      v_scale,
                      table + static_cast<int64_t>(b0) * table_width,
                      lengths + b0,
                      batch - b0 < per_launch ? batch - b0 : per_launch,
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
    const cudaError_t e = head_dim == 64 ? launch_dim<64>(a, e4m3, sms, st)
                                         : launch_dim<128>(a, e4m3, sms, st);
    if (e != cudaSuccess) return status_of(e);
  }
  return SL_OK;
}

extern "C" int sl_paged_attention_with(const sl_paged_attention_args* a) {
  if (a == nullptr) return SL_INVALID_ARG;
  return sl_paged_attention(a->q, a->k_cache, a->v_cache, a->k_scale, a->v_scale, a->cache_type, a->table, a->lengths, a->batch,
                            a->heads, a->kv_heads, a->head_dim, a->table_width, a->pages, a->page_size, a->scale, a->out, a->lse,
                            a->workspace, a->workspace_bytes, a->stream);
}
