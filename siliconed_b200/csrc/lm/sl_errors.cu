// The library's error word, one per device.
#include "sl_common.cuh"

namespace {
__device__ int g_errors[4];
}

namespace sl {

int* error_word() {
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_errors) != cudaSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  return static_cast<int*>(p);
}

}  // namespace sl

extern "C" int sl_errors(int* site) {
  int h[4] = {0, 0, 0, 0};
  const int zero[4] = {0, 0, 0, 0};
  if (site != nullptr) *site = 0;
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(h, g_errors, sizeof h) != cudaSuccess ||
      (h[0] != 0 && cudaMemcpyToSymbol(g_errors, zero, sizeof zero) != cudaSuccess)) {
    cudaGetLastError();
    return SL_CUDA_ERROR;
  }
  if (site != nullptr) *site = h[1];
  return h[0] == sc::kErrTimeout ? SL_TIMEOUT : h[0];
}
