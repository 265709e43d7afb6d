// The product of e4m3 activations and an e4m3 weight, each with fp32 scales per block of 128 (sl_linear_block_fp8).
//
//   y[i, j] = sum_b sa[i, b] sw[j / 128, b] (sum_{k in block b} a[i, k] w[j, k]) (+ bias[j])
//
// The scales change every 128 values of K, so an accumulator cannot run over all of K: the tensor cores produce one
// block's partial product in TMEM (tcgen05.mma kind::f8f6f4, four MMAs of K 32), and the epilogue warps multiply it
// by its scales and add it to fp32 sums in registers while the MMAs of the next block run into the other TMEM buffer.
//
// Two kernels, by their estimated times (swap_plan(), pair_plan()):
//
// - linear_pair: a cluster of two CTAs owns tiles of 256 x 256 of y (tcgen05.mma.cta_group::2), persistent over the
//   tiles.  Each CTA loads its own 128 rows of a and of w by TMA (128-byte swizzle).  The tile leaves through shared
//   memory by TMA stores, which run under the next tile's blocks.  What bounds it is a block's round trip through its TMEM
//   buffer: 4 MMAs (650 cycles beside the epilogue's work), their commit (350), the partial read by 16 warps (450) and the
//   buffer's release to the MMA threads (400), some 1900 cycles for the two buffers that 256 columns leave.  [4096, 3840] x
//   [3840, 10240]: 172 us, 1870 TFLOP/s in a chain of calls (191 to 205 with new inputs in every call); without the epilogue's
//   arithmetic 134 us, the loads take less.  (Beside an earlier form's 182: tiles of 256 x 128 with four buffers 198 us, their MMAs read
//   shared memory half again as often; fma.rn.f32x2 for the sums 293, pairs of registers moved together; one issuing
//   thread 212; the two halves of the columns issued by a thread each, two buffers each, 5 % slower, a is read twice; 16
//   epilogue warps of 64 columns 258, spills.)  Where the tiles leave pairs idle, a cluster of up to 4 pairs shares a
//   tile's K and adds its parts as below: [512, 9728] x [9728, 2560] 24.7 us, 46.3 without.
// - linear_swap: for few rows, bound by reading the weight.  The operands change places: 128 weight rows are the MMA's
//   M and the rows of a, in tiles of up to 64, its N, so that no MMA row or TMEM column is padding; K is cut over the
//   CTAs of a cluster, whose partials meet through distributed shared memory and are added in rank order.  The weight's
//   first tiles are prefetched to L2 while the kernel before this one ends.  One row of [4096, 12288] (from HBM, calls after
//   one another): 12.1 us, 4.2 TB/s (0.65 of a copy's rate): its begin, the cluster's join and its end take some 4 us, and 192
//   equal CTAs on 148 SMs leave 44 SMs with twice the others' bytes.  64 rows of it 17.0 us, 131 rows of [2560, 9728] 12.9 us:
//   the weight passes through shared memory once for each tile of rows, three times, 228 equal CTAs lie unevenly on the SMs, and
//   a block's chain of commit, TMEM read and sums in four warps is waited for; no resource is full (issue slots 35 %, tensor
//   pipe 12 %).  Eight epilogue warps spill and are slower.  (Room for a third
//   CTA an SM, so that the next call's begin early: 15.4 us for one row, the CTAs spread unevenly.)
//
// Rows past m or n and values past k arrive as zeros.  Every wait is bounded; no load uses cluster multicast.
#include <atomic>
#include <cmath>

#include "sl_common.cuh"

namespace sl {
namespace {

constexpr int BK = 128;         // values of K under one scale: a stage, 128 bytes a row
constexpr int kRowBytes = BK;

// kind::f8f6f4 with e4m3 operands, both K-major, fp32 accumulation.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <bool kPair>
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  if (kPair)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Waits for this thread's TMEM loads; the values it loaded cannot be used above it.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

__device__ __forceinline__ void tmem_wait(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
// 32 consecutive fp32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) { sc::tmem_ld_32(taddr, r); }
// 16 (32) consecutive columns of 16 TMEM lanes, a warp's tile: a thread gets, of every 8 columns c and of the lanes from
// `taddr` on, those of lane l / 4 in columns c + l % 4 * 2 and the next, and of lane l / 4 + 8 the same.
__device__ __forceinline__ void tmem_load_tile(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_load_tile(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kLeft) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// A barrier of the cluster's threads.  The instructions are the aligned ones, which all of a warp must reach together: lanes
// that a loop or a guarded store parted come together first.
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  sc::cluster_barrier();
}

__device__ __forceinline__ float bias_at(const uint16_t* bias, int col, int n) {
  return bias != nullptr && col < n ? from_bf16(bias[col]) : 0.0f;
}

// ------------------------------------------------------------------------------------------ many rows

namespace pair {

constexpr int BM = 128;                   // rows of a per CTA, 256 a pair
constexpr int BN = 256, BNH = BN / 2;     // columns of a pair tile; rows of w each CTA loads
constexpr int kStages = 5;
constexpr int kTileBytes = BM * kRowBytes;
constexpr int kEpiWarp0 = 4, kEpiWarps = 8;
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;
// Registers a thread after the split: the sums (128), three loads (96) and addresses; the TMA and MMA warps'
// group gives up what it does not need.  The launch checks that the kernel was built with at least their sum.
constexpr int kEpiRegisters = 232, kOtherRegisters = 40;
constexpr int kLaunchRegisters = (kOtherRegisters + 2 * kEpiRegisters + 2) / 3;
constexpr uint32_t kTmemCols = 512;       // two partial products of 256 columns
constexpr int kBoxBytes = 32 * 128;       // 32 rows of 128 bytes of y: a TMA store
constexpr int kPartRow = BN * 4;          // a row of a part's sums
constexpr int kMostParts = 4;             // pairs of a cluster

struct __align__(1024) Smem {
  uint8_t a[kStages][kTileBytes];
  uint8_t w[kStages][kTileBytes];
  uint8_t out[kEpiWarps][2][kBoxBytes];
  uint64_t full[kStages];                  // the leader's: both CTAs' bytes of the stage landed
  uint64_t done[kStages];                  // the stage's MMAs completed: its partial is there, the stage is free
  uint64_t part_empty[2];                  // the leader's: both CTAs' epilogues have read the buffer
  uint64_t drain[2];
  uint32_t tmem_base;
  int abort;
};
constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
static_assert(BM * kPartRow <= 2 * kStages * kTileBytes, "a part's sums fit the stages");

// kTmaOut: y's rows start on 16 bytes, so that whole boxes leave by TMA.
template <bool kF32Out, bool kTmaOut>
__global__ void __launch_bounds__(kThreads, 1)
    linear_pair(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                const __grid_constant__ CUtensorMap tm_y, const float* a_scales,
                const float* w_scales, const uint16_t* bias, void* y, int m, int n,
                int k_blocks, int m_tiles, int n_tiles, int parts, int* err) {
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cluster_rank = sc::cluster_ctarank(), rank = cluster_rank & 1u, lead = cluster_rank & ~1u;
  const bool leader = rank == 0;
  // `parts` pairs, a cluster, share a tile's K; above one part every cluster has one tile.
  const int part = static_cast<int>(cluster_rank >> 1);
  const int first = static_cast<int>(blockIdx.x) / (2 * parts), pairs = static_cast<int>(gridDim.x) / (2 * parts), tiles = m_tiles * n_tiles;
  const int kb0 = part * k_blocks / parts, kb1 = (part + 1) * k_blocks / parts;
  volatile int* abort = &s.abort;
  sc::pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      sc::mbar_init(&s.full[i], 1);
      sc::mbar_init(&s.done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      sc::mbar_init(&s.part_empty[i], 2 * kEpiWarps);
      sc::mbar_init(&s.drain[i], 1);
    }
    s.abort = 0;
    sc::fence_mbar_init();
    sc::prefetch_tensormap(&tm_a);
    sc::prefetch_tensormap(&tm_w);
    if (kTmaOut) sc::prefetch_tensormap(&tm_y);
  }
  if (warp == 1) {
    sc::tmem_alloc_pair(&s.tmem_base, kTmemCols);
    sc::tmem_relinquish_pair();
  }
  __syncwarp();
  sc::tc_fence_before();
  cluster_sync();
  sc::tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  sc::pdl_wait();

  if (warp >= kEpiWarp0) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegisters));
    // One row of the tile a thread, 128 of its columns: one scale block of w.
    const int ew = warp - kEpiWarp0, quarter = warp & 3, half = ew >> 2;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * BNH;
    int buf = 0, stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = first; tile < tiles && ok; tile += pairs) {
      int mt, nt;
      sc::tile_coords(tile, m_tiles, n_tiles, mt, nt);
      const int row0 = (mt * 2 + static_cast<int>(rank)) * BM + quarter * 32, row = row0 + lane;
      const int col0 = nt * BN + half * BNH;
      // The last tile's second half may have no columns: any block's scales do.
      const float* sa = a_scales + static_cast<int64_t>(min(row, m - 1)) * k_blocks;
      const float* sw = w_scales + static_cast<int64_t>(min(col0, n - 1) / BK) * k_blocks;
      float acc[BNH];
#pragma unroll
      for (int j = 0; j < BNH; ++j) acc[j] = 0.0f;
      // The scales are asked for two blocks ahead, into registers of their own for even and odd blocks: handed from one
      // to the next they would have to arrive first (one block then took 2000 cycles instead of 750).
      const int second = min(kb0 + 1, kb1 - 1);
      float a_even = sa[kb0], w_even = sw[kb0], a_odd = sa[second], w_odd = sw[second];
      const auto add_block = [&](int kb, float& a_scale, float& w_scale) {
        if (!(ok = wait_warp(&s.done[stage], phase, abort, err, kSiteLinearSum))) return;
        sc::tc_fence_after();
        const float f = a_scale * w_scale;
        const int next = min(kb + 2, kb1 - 1);
        a_scale = sa[next];
        w_scale = sw[next];
        uint32_t r[3][32];
        const auto load = [&](int q, uint32_t(&into)[32]) { tmem_load(lanes + buf * BN + q * 32, into); };
        const auto add = [&](int q, const uint32_t(&part)[32]) {
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[q * 32 + j] = fmaf(__uint_as_float(part[j]), f, acc[q * 32 + j]);
        };
        load(0, r[0]);
        load(1, r[1]);
        load(2, r[2]);
        tmem_wait(r[0]);
        tmem_wait(r[1]);
        tmem_wait(r[2]);
        add(0, r[0]);
        load(3, r[0]);
        tmem_wait(r[0]);
        // All of the partial is in registers: its buffer is free.
        sc::tc_fence_before();
        __syncwarp();
        if (lane == 0) sc::mbar_arrive_cluster(sc::peer_addr(&s.part_empty[buf], lead));
        add(1, r[1]);
        add(2, r[2]);
        add(3, r[0]);
        buf ^= 1;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      };
      for (int kb = kb0; kb < kb1 && ok; kb += 2) {
        add_block(kb, a_even, w_even);
        if (kb + 1 < kb1 && ok) add_block(kb + 1, a_odd, w_odd);
      }
      if (!ok) break;
      if (parts > 1) {
        // The sums over the stages, which nothing reads or writes any more: a row of 256 floats a thread and its neighbour
        // half, 16-byte chunks exchanged so that 8 lanes' writes meet different banks.
        uint8_t* mine = s.a[0] + (quarter * 32 + lane) * kPartRow;
#pragma unroll
        for (int q = 0; q < BNH / 4; ++q)
          *reinterpret_cast<float4*>(mine + ((half * (BNH / 4) + (q ^ (lane & 7))) << 4)) =
              make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
      } else if (kTmaOut) {
        constexpr int kBoxCols = kF32Out ? 32 : 64;  // 128 bytes
        uint8_t* out = &s.out[ew][0][0];
#pragma unroll
        for (int b = 0; b < BNH / kBoxCols; ++b) {
          if (lane == 0) bulk_wait_read<1>();  // the store of two boxes ago has read this half
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint4 v;
            if (kF32Out) {
              const int j = b * 32 + q * 4;
              v = make_uint4(__float_as_uint(acc[j] + bias_at(bias, col0 + j, n)), __float_as_uint(acc[j + 1] + bias_at(bias, col0 + j + 1, n)),
                             __float_as_uint(acc[j + 2] + bias_at(bias, col0 + j + 2, n)), __float_as_uint(acc[j + 3] + bias_at(bias, col0 + j + 3, n)));
            } else {
              float x[8];
#pragma unroll
              for (int t = 0; t < 8; ++t) x[t] = acc[b * 64 + q * 8 + t] + bias_at(bias, col0 + b * 64 + q * 8 + t, n);
              v = pack8(x);
            }
            *reinterpret_cast<uint4*>(out + (b & 1) * kBoxBytes + lane * 128 + ((q ^ (lane & 7)) << 4)) = v;
          }
          sc::fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            if (row0 < m && col0 + b * kBoxCols < n)
              tma_store_2d(&tm_y, sc::smem_u32(out + (b & 1) * kBoxBytes), col0 + b * kBoxCols, row0);
            bulk_commit();
          }
        }
      } else {
        // Rows that do not start on 16 bytes: through shared memory all the same, so that a warp's stores are of neighbours.
        // (Every lane along its own row: 178 us for [2000, 9728] x [9728, 2567], this way 94; 88 for 2560 columns.)
        constexpr int kPassCols = kF32Out ? 64 : 128, kPer = kF32Out ? 4 : 8;  // 256 bytes of a row; values of 16 bytes
        uint8_t* out = &s.out[ew][0][0];
        const int rows = min(32, m - row0);
#pragma unroll
        for (int b = 0; b < BNH / kPassCols; ++b) {
          const int col = col0 + b * kPassCols;
          __syncwarp();  // the pass before has been read
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            float x[8];
#pragma unroll
            for (int t = 0; t < kPer; ++t) x[t] = acc[b * kPassCols + q * kPer + t] + bias_at(bias, col + q * kPer + t, n);
            const uint4 v = kF32Out ? make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]))
                                    : pack8(x);
            *reinterpret_cast<uint4*>(out + lane * 256 + ((q & 8 | ((q & 7) ^ (lane & 7))) << 4)) = v;
          }
          __syncwarp();
          const auto leave = [&](auto unit) {
            using T = decltype(unit);
            constexpr int kUnits = 256 / sizeof(T), kChunk = 16 / sizeof(T), kValues = kF32Out ? 1 : sizeof(T) / 2;
            for (int t = 0; t < rows; ++t) {
              T* to = reinterpret_cast<T*>(static_cast<uint8_t*>(y) + (static_cast<int64_t>(row0 + t) * n + col) * (kF32Out ? 4 : 2));
#pragma unroll
              for (int u = lane; u < kUnits; u += 32) {
                const int chunk = u / kChunk;
                if (col + u * kValues < n)
                  to[u] = reinterpret_cast<const T*>(out + t * 256 + ((chunk & 8 | ((chunk & 7) ^ (t & 7))) << 4))[u % kChunk];
              }
            }
          };
          if (kF32Out || n % 2 == 0)
            leave(uint32_t{});
          else
            leave(uint16_t{});
        }
      }
    }
    if (kTmaOut && lane == 0) bulk_wait_all();
    if (parts > 1) {
      // Every part's pair adds a share of the rows, in the parts' order: the same sums whichever adds them.
      cluster_sync();
      int mt, nt;
      sc::tile_coords(first, m_tiles, n_tiles, mt, nt);
      const int row0 = (mt * 2 + static_cast<int>(rank)) * BM;
      const int lo = part * BM / parts, hi = (part + 1) * BM / parts;
      for (int t = lo + ew; t < hi && row0 + t < m; t += kEpiWarps)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int u = h * 32 + lane, col = nt * BN + 4 * u;
          const uint8_t* from = s.a[0] + t * kPartRow + (((u & ~7) | ((u & 7) ^ (t & 7))) << 4);
          float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int q = 0; q < parts; ++q) {
            float4 v;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                         : "r"(sc::peer_addr(from, 2 * q + rank))
                         : "memory");
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
          }
          const float out[4] = {sum.x + bias_at(bias, col, n), sum.y + bias_at(bias, col + 1, n), sum.z + bias_at(bias, col + 2, n),
                                sum.w + bias_at(bias, col + 3, n)};
          const int64_t at = static_cast<int64_t>(row0 + t) * n + col;
          if (kTmaOut) {  // n a multiple of 4 at least
            if (col < n) {
              if (kF32Out)
                *reinterpret_cast<float4*>(static_cast<float*>(y) + at) = make_float4(out[0], out[1], out[2], out[3]);
              else
                *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(y) + at) = make_uint2(pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3]));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < n) {
                if (kF32Out)
                  static_cast<float*>(y)[at + e] = out[e];
                else
                  static_cast<__nv_bfloat16*>(y)[at + e] = __float2bfloat16_rn(out[e]);
              }
          }
        }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == 0) {
      // TMA: each CTA its own halves, both CTAs' bytes counted on the leader's barrier.
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0, issued = 0, last_parity = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += pairs) {
          int mt, nt;
          sc::tile_coords(tile, m_tiles, n_tiles, mt, nt);
          const int row0 = (mt * 2 + static_cast<int>(rank)) * BM, col0 = nt * BN + static_cast<int>(rank) * BNH;
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!wait(&s.done[stage], phase ^ 1u, abort, err, kSiteLinearLoad)) {
              ok = false;
              break;
            }
            if (leader) sc::mbar_arrive_expect_tx(&s.full[stage], 4 * kTileBytes);
            const uint32_t bar = sc::peer_addr(&s.full[stage], lead);
            sc::tma_load_2d_pair(s.a[stage], &tm_a, bar, kb * BK, row0);
            sc::tma_load_2d_pair(s.w[stage], &tm_w, bar, kb * BK, col0);
            issued |= 1u << stage;
            last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        if (leader)
          for (int st = 0; st < kStages; ++st)
            if (issued & (1u << st)) sc::mbar_wait_drain(&s.full[st], (last_parity >> st) & 1u);
      }
    } else if (warp <= 2) {
      // Two threads issue the MMAs, block by block in turns, each into its own TMEM buffer: one's commit and waits (some
      // 400 cycles a block) run under the other's MMAs.
      if (leader && lane == 0) {
        constexpr uint32_t idesc = idesc_e4m3(2 * BM, BN);
        const int buf = warp - 1;
        const int blocks = (tiles - first + pairs - 1) / pairs * (kb1 - kb0);  // of this pair's tiles
        int stage = buf;
        uint32_t phase = 0, buf_phase = 0;
        for (int g = buf; g < blocks; g += 2) {
          if (!wait(&s.part_empty[buf], buf_phase ^ 1u, abort, err, kSiteLinearBuffer) ||
              !wait(&s.full[stage], phase, abort, err, kSiteLinearMma))
            break;
          sc::tc_fence_after();
          const uint32_t a0 = sc::smem_u32(s.a[stage]), b0 = sc::smem_u32(s.w[stage]);
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk)
            mma_e4m3<true>(tmem + static_cast<uint32_t>(buf * BN), sc::umma_desc_sw128(a0 + kk * 32),
                           sc::umma_desc_sw128(b0 + kk * 32), idesc, kk != 0 ? 1u : 0u);
          sc::tc_commit_pair_both(&s.done[stage], static_cast<uint16_t>(0x3u << lead));
          buf_phase ^= 1u;
          stage += 2;
          if (stage >= kStages) {
            stage -= kStages;
            phase ^= 1u;
          }
        }
        sc::tc_commit_pair(sc::peer_addr(&s.drain[buf], lead));
        sc::mbar_wait_drain(&s.drain[buf], 0);
      }
    }
    __syncwarp();
    if (parts > 1) cluster_sync();
  }
  // No CTA leaves while the pair's MMAs, TMEM or barriers or the cluster's sums may still reach its memory.
  __syncwarp();
  sc::tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    sc::tc_fence_after();
    sc::tmem_dealloc_pair(tmem, kTmemCols);
  }
}

}  // namespace pair

// ------------------------------------------------------------------------------------------ few rows

namespace swap {

constexpr int BN = 128;                   // rows of w (columns of y) a CTA
constexpr int kMostRows = 64;            // rows of a, the MMA's N
constexpr int kWBytes = BN * kRowBytes;
constexpr int kRingBytes = 100 * 1024;    // two CTAs an SM
constexpr int kMostStages = kRingBytes / (kWBytes + 16 * kRowBytes);  // 5: of 16 rows, and of 32; 4 of 48 and 64
constexpr int kGroup = 8;                 // blocks whose factors are brought in together
constexpr int kBuffers = 4;               // partial products in TMEM
constexpr int kEpiWarp0 = 3, kEpiWarps = 4, kEpiThreads = kEpiWarps * 32;
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;

struct Control {
  uint64_t full[kMostStages];
  uint64_t done[kMostStages];             // the stage's MMAs completed: its partial is there, the stage is free
  uint64_t part_empty[kBuffers];
  uint64_t drain[2];
  uint32_t tmem_base;
  int abort;
  alignas(16) float factors[2][kGroup][kMostRows];  // sa * sw of a group of blocks, by the group's parity
};
constexpr size_t kSmemBytes = kRingBytes + 1024;
static_assert(kEpiThreads == BN, "a thread per column");
static_assert(kMostRows * BN * 4 <= kRingBytes, "a partial fits the ring");
// Every wait's parity tells one phase from the next as long as nobody is two phases ahead: the MMAs of block g wait for
// the epilogue to have read block g - kBuffers, so a stage must not come round sooner than a buffer.
static_assert(kRingBytes / (kWBytes + kMostRows * kRowBytes) >= kBuffers, "stages for the buffers");

// Where column `col` of row `row` stands in shared memory.
__device__ __forceinline__ int spread(int row, int col) { return col ^ (row >> 1 & 3) << 3; }

// kRows: the sums' registers (16, 32 or 64); `rows` <= kRows is the tile's count, a multiple of 16, and the rows of
// a's TMA box.
template <bool kF32Out, int kRows>
__global__ void __launch_bounds__(kThreads, 2)
    linear_swap(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                const float* a_scales, const float* w_scales,
                const uint16_t* bias, void* y, int m, int n, int k_blocks, int rows, int stages,
                int* err) {
  constexpr uint32_t kTmemCols = kBuffers * kRows;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Control s;
  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = kWBytes + rows * kRowBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = sc::cluster_ctarank();
  uint32_t parts;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
  const int tile = static_cast<int>(blockIdx.x / parts), n0 = tile * BN, m0 = blockIdx.y * rows;
  const int kb0 = static_cast<int>(rank * static_cast<uint32_t>(k_blocks) / parts);
  const int kb1 = static_cast<int>((rank + 1) * static_cast<uint32_t>(k_blocks) / parts);
  volatile int* abort = &s.abort;
  sc::pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      sc::mbar_init(&s.full[i], 1);
      sc::mbar_init(&s.done[i], 1);
    }
    for (int i = 0; i < kBuffers; ++i) sc::mbar_init(&s.part_empty[i], kEpiWarps);
    for (int i = 0; i < 2; ++i) sc::mbar_init(&s.drain[i], 1);
    s.abort = 0;
    sc::fence_mbar_init();
    sc::prefetch_tensormap(&tm_a);
    sc::prefetch_tensormap(&tm_w);
  }
  if (warp == 1) {
    sc::tmem_alloc(&s.tmem_base, kTmemCols);
    sc::tmem_relinquish();
  }
  // The ring's first blocks of the weight on their way to L2 while the kernel before this one ends: L2 holds what that
  // kernel writes too, so nothing stale can come of it.  (All of the CTA's blocks at once: 13.0 us instead of 11.9 for one row
  // of [4096, 12288], 11.9 instead of 11.7 without any.)
  if (warp == kEpiWarp0 && lane == 0)
    for (int kb = kb0; kb < kb1 && kb < kb0 + stages; ++kb)
      asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(&tm_w)),
                   "r"(kb * BK), "r"(n0)
                   : "memory");
  sc::tc_fence_before();
  __syncthreads();
  sc::tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  sc::pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, last_parity = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!wait(&s.done[stage], phase ^ 1u, abort, err, kSiteLinearLoad)) break;
        sc::mbar_arrive_expect_tx(&s.full[stage], stage_bytes);
        sc::tma_load_2d(ring + stage * stage_bytes, &tm_w, &s.full[stage], kb * BK, n0);
        sc::tma_load_2d(ring + stage * stage_bytes + kWBytes, &tm_a, &s.full[stage], kb * BK, m0);
        issued |= 1u << stage;
        last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      for (int st = 0; st < stages; ++st)
        if (issued & (1u << st)) sc::mbar_wait_drain(&s.full[st], (last_parity >> st) & 1u);
    }
  } else if (warp < kEpiWarp0) {
    // Two threads issue the MMAs, block by block in turns: a block costs its thread some 770 cycles of issue, commit and
    // waits, its MMAs 64 to 256.
    if (lane == 0) {
      const uint32_t idesc = idesc_e4m3(BN, rows);
      const int turn = warp - 1;
      for (int g = turn; g < kb1 - kb0; g += 2) {
        const int buf = g % kBuffers, stage = g % stages;
        if (!wait(&s.part_empty[buf], (g / kBuffers & 1) ^ 1u, abort, err, kSiteLinearBuffer) ||
            !wait(&s.full[stage], g / stages & 1, abort, err, kSiteLinearMma))
          break;
        sc::tc_fence_after();
        const uint32_t w0 = sc::smem_u32(ring + stage * stage_bytes), a0 = w0 + kWBytes;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk)
          mma_e4m3<false>(tmem + static_cast<uint32_t>(buf * kRows), sc::umma_desc_sw128(w0 + kk * 32),
                          sc::umma_desc_sw128(a0 + kk * 32), idesc, kk != 0 ? 1u : 0u);
        sc::tc_commit(&s.done[stage]);
      }
      sc::tc_commit(&s.drain[turn]);
      sc::mbar_wait_drain(&s.drain[turn], 0);
    }
  } else {
    // 4 columns of y a thread and a quarter of the rows.  The factors sa * sw come through shared memory, a group of blocks
    // ahead of their use: thread t brings those of row t, lane i the weight's scale of block i.  (A column a thread and all
    // rows: every thread reads all the factors, 13.9 us for 131 rows of [2560, 9728] where this takes
    // 12.9; more columns or factors on their way at once 14.0 to 14.8.)
    const int et = threadIdx.x - kEpiWarp0 * 32, quarter = warp & 3;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const float* sw = w_scales + static_cast<int64_t>(tile) * k_blocks;
    const bool owns = et < rows && m0 + et < m;
    const float* sa = a_scales + static_cast<int64_t>(owns ? m0 + et : 0) * k_blocks;
    // Rows 8 g + l % 4 * 2 (+ 1), columns h * 16 + l / 4 (+ 8) of the warp's 32: sums [g][h][column * 2 + row].
    float acc[kRows / 8][2][4], a_next[kGroup], w_next;
#pragma unroll
    for (int j = 0; j < kRows; ++j) acc[j / 8][j / 4 % 2][j % 4] = 0.0f;
    const auto ask = [&](int kb) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) a_next[i] = owns && kb + i < kb1 ? sa[kb + i] : 0.0f;
      w_next = lane < kGroup && kb + lane < kb1 ? sw[kb + lane] : 0.0f;
    };
    ask(kb0);
    int buf = 0, stage = 0;
    uint32_t phase = 0;
    // A wait that gave up leaves the sums as they are, but the loop goes on, so that every warp meets the others at each
    // group's barrier.
    for (int kb = kb0; kb < kb1; ++kb) {
      const int in_group = (kb - kb0) % kGroup;
      float(*factors)[kMostRows] = s.factors[(kb - kb0) / kGroup & 1];
      if (in_group == 0) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          const float f = a_next[i] * __shfl_sync(0xFFFFFFFFu, w_next, i);
          if (et < kRows) factors[i][et] = f;
        }
        ask(kb + kGroup);
        sc::named_barrier_sync(1, kEpiThreads);
      }
      const float2* f = reinterpret_cast<const float2*>(factors[in_group]) + lane % 4;
      const bool ok = wait_warp(&s.done[stage], phase, abort, err, kSiteLinearSum);
      sc::tc_fence_after();
      if (ok) {
        constexpr int kChunk = kRows == 32 ? 32 : 16;  // 64 rows: the registers take no more
#pragma unroll
        for (int q = 0; q < kRows; q += kChunk) {
          if (q >= rows) break;
          uint32_t r[2][kChunk / 2];
          tmem_load_tile(lanes + buf * kRows + q, r[0]);
          tmem_load_tile(lanes + (16u << 16) + buf * kRows + q, r[1]);
          float2 v[kChunk / 8];
#pragma unroll
          for (int g = 0; g < kChunk / 8; ++g) v[g] = f[(q / 8 + g) * 4];
          tmem_wait(r[0]);
          tmem_wait(r[1]);
          if (q + kChunk >= rows) {  // all of the partial is in registers: its buffer is free
            sc::tc_fence_before();
            __syncwarp();
            if (lane == 0) sc::mbar_arrive(&s.part_empty[buf]);
          }
#pragma unroll
          for (int g = 0; g < kChunk / 8; ++g)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float& sum = acc[q / 8 + g][e / 4][e % 4];
              sum = fmaf(__uint_as_float(r[e / 4][g * 4 + e % 4]), e % 2 == 0 ? v[g].x : v[g].y, sum);
            }
        }
      }
      buf = buf + 1 == kBuffers ? 0 : buf + 1;
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // In shared memory a row's columns are exchanged in groups of 8, so that a warp's 4 rows meet different banks.
    const auto each = [&](auto&& put) {
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int g = j / 8, h = j / 4 % 2, e = j % 4;
        const int row = g * 8 + lane % 4 * 2 + e % 2, col = quarter * 32 + h * 16 + lane / 4 + e / 2 * 8;
        if (g * 8 < rows) put(row * BN + spread(row, col), acc[g][h][e], h * 2 + e / 2);
      }
    };
    if (parts == 1) {
      // Through shared memory (over the ring, as below), so that a warp's stores are of neighbours.  (Two bytes a lane straight
      // from the registers: 3900 cycles for 48 rows.)
      float add[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) add[c] = bias_at(bias, n0 + quarter * 32 + lane / 4 + c * 8, n);
      constexpr int kSize = kF32Out ? 4 : 2, kPer = 16 / kSize;  // bytes of a value, values of 16 bytes
      each([&](int at, float sum, int c) {
        if (kF32Out)
          reinterpret_cast<float*>(ring)[at] = sum + add[c];
        else
          reinterpret_cast<__nv_bfloat16*>(ring)[at] = __float2bfloat16_rn(sum + add[c]);
      });
      sc::named_barrier_sync(1, kEpiThreads);
      const int live = min(rows, m - m0);
      const bool wide = n % kPer == 0;  // rows of y start on 16 bytes
      if (wide) {
        for (int i = et; i < live * (BN / kPer); i += kEpiThreads) {
          const int t = i / (BN / kPer), c = i % (BN / kPer) * kPer;
          if (n0 + c < n)
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(y) + (static_cast<int64_t>(m0 + t) * n + n0 + c) * kSize) =
                *reinterpret_cast<const uint4*>(ring + (t * BN + spread(t, c)) * kSize);
        }
      } else if (n0 + et < n) {  // a value a lane, a row a step
#pragma unroll 1
        for (int t = 0; t < live; ++t) {
          const int64_t at = static_cast<int64_t>(m0 + t) * n + n0 + et;
          if (kF32Out)
            static_cast<float*>(y)[at] = reinterpret_cast<const float*>(ring)[t * BN + spread(t, et)];
          else
            static_cast<uint16_t*>(y)[at] = reinterpret_cast<const uint16_t*>(ring)[t * BN + spread(t, et)];
        }
      }
    } else {
      // Over the ring: every copy has arrived and every MMA has read it, or the wait for the last partial gave up and
      // the kernel's error says so.
      each([&](int at, float sum, int) { reinterpret_cast<float*>(ring)[at] = sum; });
    }
  }
  __syncwarp();
  sc::tc_fence_before();
  if (parts > 1) {
    // Every CTA adds a share of the rows, in rank order: the same sums whichever CTA adds them.  (The warps are together; a
    // second __syncwarp() here: 12.3 us for one row of [4096, 12288], 12.05 without.)
    sc::cluster_barrier();
    const int cp = threadIdx.x % (BN / 2), group = threadIdx.x / (BN / 2);
    const int lo = static_cast<int>(rank) * rows / static_cast<int>(parts), hi = static_cast<int>(rank + 1) * rows / static_cast<int>(parts);
    const int col = n0 + 2 * cp;
    const float b0 = bias_at(bias, col, n), b1 = bias_at(bias, col + 1, n);
    const bool both = n % 2 == 0 && col + 1 < n;
    constexpr int kAdders = kThreads / (BN / 2);  // whole groups of threads
    for (int t = lo + group; group < kAdders && t < hi && m0 + t < m; t += kAdders) {
      const float* mine = reinterpret_cast<const float*>(ring) + t * BN + spread(t, 2 * cp);
      float2 sum = make_float2(0.0f, 0.0f);
      for (uint32_t q = 0; q < parts; ++q) {
        float2 v;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(sc::peer_addr(mine, q)) : "memory");
        sum.x += v.x;
        sum.y += v.y;
      }
      sum.x += b0;
      sum.y += b1;
      const int64_t at = static_cast<int64_t>(m0 + t) * n + col;
      if (kF32Out) {
        float* o = static_cast<float*>(y) + at;
        if (both) {
          *reinterpret_cast<float2*>(o) = sum;
        } else {
          if (col < n) o[0] = sum.x;
          if (col + 1 < n) o[1] = sum.y;
        }
      } else {
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(y) + at;
        if (both) {
          *reinterpret_cast<uint32_t*>(o) = pack_bf16x2(sum.x, sum.y);
        } else {
          if (col < n) o[0] = __float2bfloat16_rn(sum.x);
          if (col + 1 < n) o[1] = __float2bfloat16_rn(sum.y);
        }
      }
    }
    cluster_sync();  // the partials stay until the other CTAs have read them
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    sc::tc_fence_after();
    sc::tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace swap

// ------------------------------------------------------------------------------------------ the launch

typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

encode_fn encoder() {
  static const encode_fn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<encode_fn>(p);
  }();
  return fn;
}

// A row-major [rows][cols] matrix in boxes of 128 bytes x `box` rows, 128-byte swizzle, zeros outside.
bool make_map(CUtensorMap* map, encode_fn enc, CUtensorMapDataType type, int size, const void* base, int64_t rows, int64_t cols,
              int box) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * size};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(128 / size), static_cast<cuuint32_t>(box)};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Product {
  const uint8_t *a, *w;
  const float *a_scales, *w_scales;
  const uint16_t* bias;
  int64_t m, n, k;
  void* y;
  bool f32;
  int k_blocks, sms;
  encode_fn enc;
  int* err;
  cudaStream_t stream;
};

template <typename... Params, typename... Args>
cudaError_t launch_cluster(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream,
                           Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Kernels that never run, with the two kernels' threads and room: what the runtime says of them holds for those, of which it
// would count one CTA an SM because they allocate TMEM (of the few-rows kernel two fit).
__global__ void __launch_bounds__(swap::kThreads, 2) seat_swap() {}
__global__ void __launch_bounds__(pair::kThreads, 1) seat_pair() {}

// How many CTAs run at once in clusters of `c`.  A cluster lies in one group of SMs, so most sizes leave slots empty: for the
// few-rows kernel, two CTAs an SM, 148 SMs hold 296 CTAs in clusters of 2, 279 of 3, 284 of 4, 280, 270, 259 and 264 of 5 to
// 8, and the first CTA past that starts a second wave (one row, k 5120 to 10240: 10.5 us up to 284 in clusters of 4,
// 14.8 from 288).  The runtime is asked once per device and size.  0: it gave an error.
template <bool kPair>
int cluster_capacity(int c, int dev) {
  static std::atomic<int> known[64][9];
  if (dev < 64)
    if (const int n = known[dev][c].load(std::memory_order_relaxed); n != 0) return n;
  static unsigned long long configured = 0;
  constexpr size_t kRoom = kPair ? pair::kSmemBytes : swap::kSmemBytes + sizeof(swap::Control);
  const auto seat = kPair ? seat_pair : seat_swap;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(c));
  cfg.blockDim = dim3(kPair ? pair::kThreads : swap::kThreads);
  cfg.dynamicSmemBytes = kRoom;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(c);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (set_smem_once(seat, static_cast<int>(kRoom), configured) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, seat, &cfg) != cudaSuccess || clusters < 1) {
    cudaGetLastError();
    return 0;
  }
  if (dev < 64) known[dev][c].store(clusters * c, std::memory_order_relaxed);
  return clusters * c;
}

// Estimated microseconds with the weight in HBM, fitted (B200) to [m, 4096] x [4096, 12288 or 4096], [m, 12288] x [12288, 4096],
// [m, 2560] x [2560, 9728 or 2560], [m, 9728] x [9728, 2560] and [m, 512] x [512, 1000], m 1 to 1024 and 1 to 8 parts; most
// within 10 %.  None of these has a long output and a short K, and neither estimate has a term for the output's bytes: [1000, 1024]
// x [1024, 7001] is estimated at 16 us and takes 25 (4.3 by its bytes and operations).  The few-rows kernel: a begin and an end, longer where a cluster adds (and then for every wave); a CTA's
// blocks one after another, slower with more rows and more CTAs an SM, so that a last wave of few CTAs is shorter; and the
// weight's bytes.  The parts this picks are the fastest or within 3 % of them.
struct SwapPlan {
  int row_tiles, rows, parts;  // parts: of K, a cluster's CTAs
  double us;
};
SwapPlan swap_plan(int64_t m, int64_t n, int k_blocks, int sms, int dev) {
  SwapPlan s;
  s.row_tiles = static_cast<int>((m + swap::kMostRows - 1) / swap::kMostRows);
  s.rows = static_cast<int>(((m + s.row_tiles - 1) / s.row_tiles + 15) / 16 * 16);
  const double n_tiles = static_cast<double>((n + swap::BN - 1) / swap::BN);
  s.parts = 1;
  s.us = 0.0;
  for (int c = 1; c <= 8 && c <= k_blocks; ++c) {
    const int room = cluster_capacity<false>(c, dev);
    if (room == 0) continue;
    const double ctas = n_tiles * s.row_tiles * c, full = std::ceil(ctas / room) - 1.0, last = ctas - full * room;
    const auto blocks = [&](double at_once) {
      return (k_blocks + c - 1) / c * (0.1 + s.rows * ((c > 1 ? 0.0058 : 0.0047) + 0.0015 * at_once / sms));
    };
    const double us = (c > 1 ? 4.2 * (full + 1.0) : 2.9) + full * blocks(room) + blocks(last) + n_tiles * k_blocks * 1.27e-3;
    if (s.us == 0.0 || us <= s.us) {
      s.us = us;
      s.parts = c;
    }
  }
  return s;
}
// The many-rows kernel: a tile's blocks one after another, and the weight's bytes.  Where the tiles leave pairs idle, a cluster
// of pairs shares each tile's K.
struct PairPlan {
  int parts;
  double us;
};
PairPlan pair_plan(int64_t m, int64_t n, int k_blocks, int sms, int dev) {
  const double n_tiles = static_cast<double>((n + pair::BN - 1) / pair::BN);
  const double tiles = static_cast<double>((m + 2 * pair::BM - 1) / (2 * pair::BM)) * n_tiles, waves = std::ceil(tiles / (sms / 2));
  const double bytes = n_tiles * k_blocks * 1.6e-3;
  PairPlan plan = {1, 6.3 + k_blocks * (0.63 * waves - 0.1) + bytes};
  for (int c = 2; c <= pair::kMostParts && c <= k_blocks && tiles * c <= sms / 2; ++c) {
    if (tiles * 2 * c > cluster_capacity<true>(2 * c, dev)) continue;
    const double us = 10.0 + (k_blocks + c - 1) / c * 0.53 + bytes;
    if (us < plan.us) plan = {c, us};
  }
  return plan;
}

template <bool kF32Out, bool kTmaOut>
cudaError_t launch_pair_as(const Product& p, int parts) {
  using namespace pair;
  auto kernel = linear_pair<kF32Out, kTmaOut>;
  static unsigned long long configured = 0;
  if (const cudaError_t e = set_smem_once(kernel, static_cast<int>(kSmemBytes), configured); e != cudaSuccess) return e;
  static const int registers = [kernel] {
    cudaFuncAttributes attr;
    return cudaFuncGetAttributes(&attr, kernel) == cudaSuccess ? attr.numRegs : 0;
  }();
  if (registers < kLaunchRegisters) return cudaErrorLaunchOutOfResources;
  CUtensorMap ta, tw, ty = {};
  if (!make_map(&ta, p.enc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.a, p.m, p.k, BM) ||
      !make_map(&tw, p.enc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.w, p.n, p.k, BNH) ||
      (kTmaOut && !make_map(&ty, p.enc, kF32Out ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                            kF32Out ? 4 : 2, p.y, p.m, p.n, 32)))
    return cudaErrorInvalidValue;
  const int m_tiles = static_cast<int>((p.m + 2 * BM - 1) / (2 * BM)), n_tiles = static_cast<int>((p.n + BN - 1) / BN);
  const int64_t tiles = static_cast<int64_t>(m_tiles) * n_tiles;
  const int clusters = static_cast<int>(parts > 1 || tiles < p.sms / 2 ? tiles : p.sms / 2);
  return launch_cluster(kernel, dim3(static_cast<unsigned>(2 * parts * clusters)), kThreads, kSmemBytes, 2 * parts, p.stream, ta, tw,
                        ty, p.a_scales, p.w_scales, p.bias, p.y, static_cast<int>(p.m), static_cast<int>(p.n), p.k_blocks, m_tiles,
                        n_tiles, parts, p.err);
}

cudaError_t launch_pair(const Product& p, int parts) {
  const bool tma = p.n % (p.f32 ? 4 : 8) == 0;
  if (p.f32) return tma ? launch_pair_as<true, true>(p, parts) : launch_pair_as<true, false>(p, parts);
  return tma ? launch_pair_as<false, true>(p, parts) : launch_pair_as<false, false>(p, parts);
}

template <bool kF32Out, int kRows>
cudaError_t launch_swap_as(const Product& p, const SwapPlan& plan) {
  using namespace swap;
  const int rows = plan.rows, parts = plan.parts;
  auto kernel = linear_swap<kF32Out, kRows>;
  static unsigned long long configured = 0;
  if (const cudaError_t e = set_smem_once(kernel, static_cast<int>(kSmemBytes), configured); e != cudaSuccess) return e;
  CUtensorMap ta, tw;
  if (!make_map(&ta, p.enc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.a, p.m, p.k, rows) ||
      !make_map(&tw, p.enc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.w, p.n, p.k, BN))
    return cudaErrorInvalidValue;
  const int64_t n_tiles = (p.n + BN - 1) / BN;
  const int stages = kRingBytes / (kWBytes + rows * kRowBytes);  // rows are 16 at least
  return launch_cluster(kernel, dim3(static_cast<unsigned>(n_tiles * parts), static_cast<unsigned>(plan.row_tiles)),
                        kThreads, kSmemBytes, parts, p.stream, ta, tw, p.a_scales, p.w_scales, p.bias, p.y,
                        static_cast<int>(p.m), static_cast<int>(p.n), p.k_blocks, rows, stages, p.err);
}

template <bool kF32Out>
cudaError_t launch_swap(const Product& p, const SwapPlan& plan) {
  return plan.rows <= 16    ? launch_swap_as<kF32Out, 16>(p, plan)
         : plan.rows <= 32  ? launch_swap_as<kF32Out, 32>(p, plan)
                            : launch_swap_as<kF32Out, 64>(p, plan);
}

}  // namespace
}  // namespace sl

extern "C" int sl_linear_block_fp8(const uint8_t* a, const float* a_scales, const uint8_t* w, const float* w_scales,
                                   const uint16_t* bias, int64_t m, int64_t n, int64_t k, void* y, int y_type,
                                   void* stream) {
  using namespace sl;
  // Tile coordinates and tile counts are 32-bit.
  if (m < 0 || m > 0x7FFFFF00 || n < 1 || n > 0x7FFFFF00 || k < 16 || k % 16 != 0 || k > 0x7FFFFF00 ||
      (m / 128 + 1) * (n / 128 + 1) > 0x0FFFFFFF || (y_type != SL_BF16 && y_type != SL_F32))
    return SL_INVALID_ARG;
  if (m == 0) return SL_OK;
  for (const void* p : {static_cast<const void*>(a), static_cast<const void*>(w), static_cast<const void*>(y)})
    if (p == nullptr || !aligned(p, 16)) return SL_INVALID_ARG;
  if (a_scales == nullptr || w_scales == nullptr || !aligned(a_scales, 4) || !aligned(w_scales, 4) || !aligned(bias, 2))
    return SL_INVALID_ARG;
  const Device device = current_device();
  const Product p{a, w, a_scales, w_scales, bias, m, n, k, y, y_type == SL_F32, static_cast<int>((k + BK - 1) / BK),
                  device.sms, encoder(), device.err, static_cast<cudaStream_t>(stream)};
  if (p.enc == nullptr || p.err == nullptr || p.sms < 2) return SL_CUDA_ERROR;
  // Up to 64 rows are always the few-rows kernel's; its row tiles are the grid's second dimension.  (Both measured, us, few-rows
  // and many-rows kernel: [m, 2560] x [2560, 9728] 14.3 and 18.3 at 192 rows, 25.3 and 18.5 at 256, 29.1 and 31.3 at 384;
  // [m, 4096] x [4096, 4096] 16.7 and 23.4 at 256, 22.1 and 19.4 at 512.)
  PairPlan many = {1, 0.0};
  if (m > swap::kMostRows) many = pair_plan(m, n, p.k_blocks, p.sms, device.index);
  if (m <= int64_t{65535} * swap::kMostRows) {
    const SwapPlan few = swap_plan(m, n, p.k_blocks, p.sms, device.index);
    if (m <= swap::kMostRows || few.us < many.us) return status_of(p.f32 ? launch_swap<true>(p, few) : launch_swap<false>(p, few));
  }
  return status_of(launch_pair(p, many.parts));
}

extern "C" int sl_linear_block_fp8_with(const sl_linear_block_fp8_args* a) {
  if (a == nullptr) return SL_INVALID_ARG;
  return sl_linear_block_fp8(a->a, a->a_scales, a->w, a->w_scales, a->bias, a->m, a->n, a->k, a->y, a->y_type, a->stream);
}
