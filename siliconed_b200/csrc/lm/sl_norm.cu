// The residual addition, RMS norm and quantization to e4m3 in blocks of 128 (sl_rms_norm_quantize).
//
//   z = x + delta;  x_out = z in x's type;  y = z * rsqrt(mean(z^2) + eps) * weight;
//   per block of 128 values of a row  s = max(max|y| / 448, 1e-30),  codes = e4m3(y / s).
//
// Bound by HBM: every value of x and delta is read once, x_out and the codes are written once.  One CTA per row
// keeps z in registers between the sum of squares and the quantization, eight consecutive values a thread and
// step (16 bytes of bf16, 32 of fp32); 16 neighbouring lanes hold one block of 128, so a block's maximum takes
// four shuffles.  Measured (B200): [4608, 3840] fp32 + fp32 38 us, 6.1 TB/s (0.94 of a copy's rate); one row of 2560
// 2.7 us in a chain of calls.
#include "sl_common.cuh"

namespace sl {
namespace {

constexpr int kMaxDim = 16384;

template <bool kF32>
__device__ __forceinline__ void load_row8(const void* row, int i, float (&v)[8]) {
  if (kF32)
    load8(static_cast<const float*>(row) + 8 * i, v);
  else
    unpack8(static_cast<const uint4*>(row)[i], v);
}

// kDelta: 0 none, 1 bf16, 2 fp32.  kVec: steps of 8 values a thread.
template <bool kF32, int kDelta, int kVec>
__global__ void __launch_bounds__(256) rms_norm_quantize_k(const void* x, const void* delta, const float* weight,
                                                           float eps, int norm, int d, void* x_out, uint8_t* codes,
                                                           float* scales) {
  __shared__ float red[8];
  sc::pdl_launch_dependents();
  sc::pdl_wait();
  const int64_t row = blockIdx.x;
  const int chunks = d / 8, blocks = (d + SL_BLOCK - 1) / SL_BLOCK;
  const char* xr = static_cast<const char*>(x) + row * d * (kF32 ? 4 : 2);
  const char* dr = static_cast<const char*>(delta) + row * d * (kDelta == 2 ? 4 : 2);
  float z[kVec][8];
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int i = threadIdx.x + j * blockDim.x;
    if (i < chunks) {
      load_row8<kF32>(xr, i, z[j]);
      if (kDelta != 0) {
        float e[8];
        load_row8<kDelta == 2>(dr, i, e);
#pragma unroll
        for (int t = 0; t < 8; ++t) z[j][t] += e[t];
        if (kF32) {
          float4* o = reinterpret_cast<float4*>(static_cast<char*>(x_out) + row * d * 4) + 2 * i;
          o[0] = make_float4(z[j][0], z[j][1], z[j][2], z[j][3]);
          o[1] = make_float4(z[j][4], z[j][5], z[j][6], z[j][7]);
        } else {
          reinterpret_cast<uint4*>(static_cast<char*>(x_out) + row * d * 2)[i] = pack8(z[j]);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) z[j][t] = 0.0f;
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) ss += z[j][t] * z[j][t];
  }
  float inv = 1.0f;
  if (norm) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, off);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = 0.0f;
    for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) ss += red[w];
    inv = 1.0f / sqrtf(ss / static_cast<float>(d) + eps);
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int i = threadIdx.x + j * blockDim.x;
    if (i - (i & 15) >= chunks) break;  // the whole block of 128 is past the row
    float y[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) y[t] = z[j][t] * inv;
    if (weight != nullptr && i < chunks) {
      float w[8];
      load8(weight + 8 * i, w);
#pragma unroll
      for (int t = 0; t < 8; ++t) y[t] *= w[t];
    }
    uint32_t m = i < chunks ? abs_max8(y) : 0u;
    const uint32_t half = 0xFFFFu << (threadIdx.x & 16);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(half, m, off));
    const float s = scale_of(m);
    if (i < chunks) reinterpret_cast<uint2*>(codes + row * d)[i] = quantize8(y, s);
    if ((i & 15) == 0) scales[row * blocks + i / 16] = s;
  }
}

template <bool kF32, int kDelta>
cudaError_t launch_norm(const void* x, const void* delta, const float* weight, float eps, int norm, int64_t rows, int d,
                        void* x_out, uint8_t* codes, float* scales, cudaStream_t stream) {
  const int chunks = d / 8;
  const int threads = chunks >= 256 ? 256 : (chunks + 31) / 32 * 32;
  const int vec = (chunks + threads - 1) / threads;
  auto kernel = vec <= 1   ? rms_norm_quantize_k<kF32, kDelta, 1>
                : vec <= 2 ? rms_norm_quantize_k<kF32, kDelta, 2>
                : vec <= 4 ? rms_norm_quantize_k<kF32, kDelta, 4>
                           : rms_norm_quantize_k<kF32, kDelta, 8>;
  return launch(kernel, dim3(static_cast<unsigned>(rows)), dim3(static_cast<unsigned>(threads)), 0, stream, x, delta,
                weight, eps, norm, d, x_out, codes, scales);
}

}  // namespace
}  // namespace sl

extern "C" int sl_rms_norm_quantize(const void* x, int x_type, const void* delta, int delta_type, const float* weight,
                                    float eps, int norm, int64_t rows, int d, void* x_out, uint8_t* codes, float* scales,
                                    void* stream) {
  using namespace sl;
  if ((x_type != SL_BF16 && x_type != SL_F32) || rows < 0 || rows > 0x7FFFFFFF || d < 16 || d > kMaxDim || d % 16 != 0)
    return SL_INVALID_ARG;
  if (delta != nullptr && delta_type != SL_BF16 && delta_type != SL_F32) return SL_INVALID_ARG;
  if (rows == 0) return SL_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr || !aligned(x, 16) || !aligned(codes, 16) ||
      !aligned(scales, 4) || !aligned(weight, 16))
    return SL_INVALID_ARG;
  if (delta != nullptr ? (x_out == nullptr || !aligned(x_out, 16) || !aligned(delta, 16))
                       : (x_out != nullptr && x_out != x))
    return SL_INVALID_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int kind = delta == nullptr ? 0 : delta_type == SL_BF16 ? 1 : 2;
  auto go = x_type == SL_F32
                ? (kind == 0 ? launch_norm<true, 0> : kind == 1 ? launch_norm<true, 1> : launch_norm<true, 2>)
                : (kind == 0 ? launch_norm<false, 0> : kind == 1 ? launch_norm<false, 1> : launch_norm<false, 2>);
  return status_of(go(x, delta, weight, eps, norm, rows, d, x_out, codes, scales, st));
}

extern "C" int sl_rms_norm_quantize_with(const sl_rms_norm_quantize_args* a) {
  if (a == nullptr) return SL_INVALID_ARG;
  return sl_rms_norm_quantize(a->x, a->x_type, a->delta, a->delta_type, a->weight, a->eps, a->norm, a->rows, a->d, a->x_out, a->codes,
                              a->scales, a->stream);
}
