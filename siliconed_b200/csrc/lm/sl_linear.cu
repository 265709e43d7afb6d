// The product of e4m3 activations and an e4m3 weight, each with fp32 scales per block of 128 (sl_linear_block_fp8).
//
//   y[i, j] = sum_b sa[i, b] sw[j / 128, b] (sum_{k in block b} a[i, k] w[j, k]) (+ bias[j])
//
// The scales change every 128 values of K, so an accumulator cannot run over all of K: the tensor cores produce one
// block's partial product in TMEM (tcgen05.mma kind::f8f6f4, four MMAs of K 32), and the epilogue warps multiply it
// by its scales and add it to fp32 sums in registers while the MMAs of the next blocks run into other TMEM buffers.
//
// One CTA per 128 x 128 tile of y.  Warp 0: TMA (a and w tiles of 128 rows x 128 bytes, 128-byte swizzle, a ring of
// kStages); warp 1: TMEM and MMA issue; warps 2-5: one row of the tile a thread.  Rows past m or n and values past k
// arrive as zeros.  Every wait is bounded; no load uses cluster multicast.
#include "sl_common.cuh"

namespace sl {
namespace {

constexpr int BM = 128, BN = 128, BK = 128;
constexpr int kStages = 5;
constexpr int kBuffers = 4;                // TMEM buffers of BN columns
constexpr int kTileBytes = BM * BK;
constexpr int kThreads = 192;
constexpr uint32_t kTmemCols = kBuffers * BN;

struct __align__(1024) Smem {
  uint8_t a[kStages][kTileBytes];
  uint8_t w[kStages][kTileBytes];
  uint64_t full[kStages], empty[kStages];
  uint64_t part_full[kBuffers], part_empty[kBuffers];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");

// kind::f8f6f4 with e4m3 operands, both K-major, fp32 accumulation.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <bool kF32Out>
__global__ void __launch_bounds__(kThreads, 1)
    linear_block_fp8_k(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w,
                       const float* __restrict__ a_scales, const float* __restrict__ w_scales,
                       const uint16_t* __restrict__ bias, void* __restrict__ y, int m, int n, int k_blocks, int* err) {
  extern __shared__ uint8_t smem_raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
  volatile int* abort = &s.abort;
  sc::pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      sc::mbar_init(&s.full[i], 1);
      sc::mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      sc::mbar_init(&s.part_full[i], 1);
      sc::mbar_init(&s.part_empty[i], 4);
    }
    sc::mbar_init(&s.drain, 1);
    s.abort = 0;
    sc::fence_mbar_init();
    sc::prefetch_tensormap(&tm_a);
    sc::prefetch_tensormap(&tm_w);
  }
  if (warp == 1) {
    sc::tmem_alloc(&s.tmem_base, kTmemCols);
    sc::tmem_relinquish();
  }
  sc::tc_fence_before();
  __syncthreads();
  sc::tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  sc::pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, last_parity = 0;
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!sc::mbar_wait(&s.empty[stage], phase ^ 1u, abort, err, kSiteLinearLoad)) break;
        sc::mbar_arrive_expect_tx(&s.full[stage], 2 * kTileBytes);
        sc::tma_load_2d(s.a[stage], &tm_a, &s.full[stage], kb * BK, m0);
        sc::tma_load_2d(s.w[stage], &tm_w, &s.full[stage], kb * BK, n0);
        issued |= 1u << stage;
        last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      for (int st = 0; st < kStages; ++st)
        if (issued & (1u << st)) sc::mbar_wait_drain(&s.full[st], (last_parity >> st) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(BM, BN);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!sc::mbar_wait(&s.part_empty[buf], buf_phase ^ 1u, abort, err, kSiteLinearBuffer) ||
            !sc::mbar_wait(&s.full[stage], phase, abort, err, kSiteLinearMma))
          break;
        sc::tc_fence_after();
        const uint32_t a0 = sc::smem_u32(s.a[stage]), b0 = sc::smem_u32(s.w[stage]);
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk)
          mma_e4m3(tmem + static_cast<uint32_t>(buf * BN), sc::umma_desc_sw128(a0 + kk * 32), sc::umma_desc_sw128(b0 + kk * 32),
                   idesc, kk != 0 ? 1u : 0u);
        sc::tc_commit(&s.empty[stage]);
        sc::tc_commit(&s.part_full[buf]);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
        if (++buf == kBuffers) {
          buf = 0;
          buf_phase ^= 1u;
        }
      }
      sc::tc_commit(&s.drain);
      sc::mbar_wait_drain(&s.drain, 0);
    }
  } else {
    const int ew = warp & 3;  // a warp reads the TMEM lanes of its rank modulo 4
    const int row = m0 + ew * 32 + lane;
    const float* sa = a_scales + static_cast<int64_t>(min(row, m - 1)) * k_blocks;
    const float* sw = w_scales + static_cast<int64_t>(blockIdx.x) * k_blocks;
    float acc[BN];
#pragma unroll
    for (int j = 0; j < BN; ++j) acc[j] = 0.0f;
    int buf = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int kb = 0; kb < k_blocks; ++kb) {
      const float f = sa[kb] * sw[kb];
      int got = 0;
      if (lane == 0) got = sc::mbar_wait(&s.part_full[buf], phase, abort, err, kSiteLinearSum) ? 1 : 0;
      ok = __shfl_sync(0xFFFFFFFFu, got, 0) != 0;
      if (!ok) break;
      sc::tc_fence_after();
#pragma unroll
      for (int q = 0; q < BN / 32; ++q) {
        uint32_t r[32];
        sc::tmem_ld_32(tmem + (static_cast<uint32_t>(ew * 32) << 16) + buf * BN + q * 32, r);
        sc::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[q * 32 + j] += f * __uint_as_float(r[j]);
      }
      sc::tc_fence_before();
      __syncwarp();
      if (lane == 0) sc::mbar_arrive(&s.part_empty[buf]);
      if (++buf == kBuffers) {
        buf = 0;
        phase ^= 1u;
      }
    }
    if (ok && row < m) {
      const int64_t at = static_cast<int64_t>(row) * n + n0;
      const bool wide = n % 8 == 0;  // rows of y start on 16 bytes
#pragma unroll
      for (int j = 0; j < BN; j += 8) {
        float v[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          v[t] = acc[j + t];
          if (bias != nullptr && n0 + j + t < n) v[t] += from_bf16(bias[n0 + j + t]);
        }
        if (wide && n0 + j < n) {
          if (kF32Out) {
            float4* o = reinterpret_cast<float4*>(static_cast<float*>(y) + at + j);
            o[0] = make_float4(v[0], v[1], v[2], v[3]);
            o[1] = make_float4(v[4], v[5], v[6], v[7]);
          } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(y) + at + j) = pack8(v);
          }
        } else if (!wide) {
#pragma unroll
          for (int t = 0; t < 8; ++t)
            if (n0 + j + t < n) {
              if (kF32Out)
                static_cast<float*>(y)[at + j + t] = v[t];
              else
                static_cast<__nv_bfloat16*>(y)[at + j + t] = __float2bfloat16_rn(v[t]);
            }
        }
      }
    }
  }
  __syncwarp();
  sc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    sc::tc_fence_after();
    sc::tmem_dealloc(tmem, kTmemCols);
  }
}

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

// [rows][k] bytes with boxes of 128 values x `box` rows, 128-byte swizzle, zeros outside.
bool make_map(CUtensorMap* map, encode_fn enc, const uint8_t* base, int64_t rows, int64_t k, int box) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(k)};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(BK), static_cast<cuuint32_t>(box)};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, boxes, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace sl

extern "C" int sl_linear_block_fp8(const uint8_t* a, const float* a_scales, const uint8_t* w, const float* w_scales,
                                   const uint16_t* bias, int64_t m, int64_t n, int64_t k, void* y, int y_type,
                                   void* stream) {
  using namespace sl;
  // Tile coordinates are 32-bit; the grid's second dimension ends at 65535 tiles.
  if (m < 0 || m > 65535LL * BM || n < 1 || n > 0x7FFFFF00 || k < 16 || k % 16 != 0 || k > 0x7FFFFF00 ||
      (y_type != SL_BF16 && y_type != SL_F32))
    return SL_INVALID_ARG;
  if (m == 0) return SL_OK;
  for (const void* p : {static_cast<const void*>(a), static_cast<const void*>(w), static_cast<const void*>(y)})
    if (p == nullptr || !aligned(p, 16)) return SL_INVALID_ARG;
  if (a_scales == nullptr || w_scales == nullptr || !aligned(a_scales, 4) || !aligned(w_scales, 4) || !aligned(bias, 2))
    return SL_INVALID_ARG;
  encode_fn enc = encoder();
  int* err = error_word();
  if (enc == nullptr || err == nullptr) return SL_CUDA_ERROR;
  CUtensorMap ta, tw;
  if (!make_map(&ta, enc, a, m, k, BM) || !make_map(&tw, enc, w, n, k, BN)) return SL_INVALID_ARG;
  auto kernel = y_type == SL_F32 ? linear_block_fp8_k<true> : linear_block_fp8_k<false>;
  if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemBytes));
      e != cudaSuccess)
    return status_of(e);
  const dim3 grid(static_cast<unsigned>((n + BN - 1) / BN), static_cast<unsigned>((m + BM - 1) / BM));
  return status_of(launch(kernel, grid, dim3(kThreads), kSmemBytes, static_cast<cudaStream_t>(stream), ta, tw, a_scales,
                          w_scales, bias, y, static_cast<int>(m), static_cast<int>(n),
                          static_cast<int>((k + BK - 1) / BK), err));
}
