// What the decoder operators share: types' loads and stores, the e4m3 block quantization, the device error
// word and the launch with programmatic stream serialization.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../sc_ptx.cuh"
#include "siliconed_lm.h"

namespace sl {

constexpr int kErrRange = SL_OUT_OF_RANGE;

// Sites recorded in the error word.
enum Site : int {
  kSiteAppendSequence = 41,
  kSiteAppendPosition = 42,
  kSiteAppendPage = 43,
  kSiteAttentionLength = 44,
  kSiteAttentionPage = 45,
  kSiteAttentionCopy = 50,
  kSiteLinearLoad = 46,
  kSiteLinearMma = 47,
  kSiteLinearBuffer = 48,
  kSiteLinearSum = 49,
};

constexpr float kE4m3Max = 448.0f;
constexpr float kScaleFloor = 1e-30f;

// What a launch needs to know of the current device, asked of the runtime once per device.
struct Device {
  int index;
  int sms;   // its SMs; 0: the runtime gave an error
  int* err;  // the library's error word: [0] the code, [1] the site, [2] the block
};
Device current_device();

inline int status_of(cudaError_t e) {
  if (e == cudaSuccess) return SL_OK;
  cudaGetLastError();
  return SL_CUDA_ERROR;
}

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// cudaFuncSetAttribute(kernel, MaxDynamicSharedMemorySize, bytes) once per kernel and device.
template <typename Kernel>
cudaError_t set_smem_once(Kernel kernel, int bytes, unsigned long long& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
  if (__atomic_load_n(&done, __ATOMIC_RELAXED) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) __atomic_fetch_or(&done, bit, __ATOMIC_RELAXED);
  return e;
}

// A launch whose set-up may overlap the end of the kernel before it on the stream.  Every kernel launched so
// executes griddepcontrol.wait in every thread before its first global access, and so orders itself after
// everything its predecessor was ordered after.  What that predecessor wrote changes while this kernel is already running, so
// no pointer is __restrict__ const and no load a read-only one (ld.global.nc): those promise values that stay the same for the
// kernel's whole life.
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Waits for the phase of `bar` with parity `parity`, as sc::mbar_wait, but without reading the global timer until many
// tries have failed: most waits here are short ones on a kernel's critical path.  Gives up (and raises `abort`) after
// sc::kWaitLimitNs.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err, int site) {
  unsigned long long since = 0;
  for (uint32_t i = 1;; ++i) {
    if (sc::mbar_try_wait(bar, parity)) return true;
    if ((i & 31u) != 0) continue;
    if (*abort) return false;
    const unsigned long long now = sc::global_ns();
    if (since == 0) since = now;
    if (now - since > sc::kWaitLimitNs) {
      sc::record_error(err, sc::kErrTimeout, site);
      *abort = 1;
      return false;
    }
  }
}

// A warp's wait: all or none.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, int* err, int site) {
  const bool got = wait(bar, parity, abort, err, site);
  return __all_sync(0xFFFFFFFFu, got) != 0;
}

__device__ __forceinline__ float from_bf16(uint32_t u) { return __uint_as_float(u << 16); }

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight consecutive values, as fp32.
__device__ __forceinline__ void unpack8(uint4 u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// Two fp32 values to e4m3 codes (nearest-even, clipped to +-448, a NaN stays NaN): `lo` in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The bits of max|v|: compared as whole numbers, so an infinity stands above every finite value and a NaN above
// that, and neither is lost.
__device__ __forceinline__ uint32_t abs_max8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

// The scale of values whose largest magnitude has the bits `m`: max(m / 448, 1e-30), a NaN or infinity as it is.  The
// quotient by the constant is a product with its reciprocal (an ulp of fp32).  With divisions here and in quantize8() the norm
// of [4608, 3840] takes 40.4 us for 38.0, one row 3.1 for 2.6 and a prompt's append to an e4m3 cache 19.1 for 17.0.
__device__ __forceinline__ float scale_of(uint32_t m) {
  return m >= 0x7F800000u ? __uint_as_float(m) : fmaxf(__uint_as_float(m) * (1.0f / kE4m3Max), kScaleFloor);
}

// Eight codes e4m3(v / s), by the reciprocal of s (an ulp of fp32; the product's rounding makes it under two).  s is at least 1e-30 and at most 7.6e35, so the
// reciprocal neither overflows nor is subnormal; a product past 448 by an ulp is clipped to it.
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return make_uint2(e4m3x2(v[0] * r, v[1] * r) | (e4m3x2(v[2] * r, v[3] * r) << 16),
                    e4m3x2(v[4] * r, v[5] * r) | (e4m3x2(v[6] * r, v[7] * r) << 16));
}

}  // namespace sl
