// The library's error word, one per device, and what is remembered of each device.
#include <atomic>

#include "sl_common.cuh"

namespace {
__device__ int g_errors[4];

constexpr int kDevices = 64;
std::atomic<int> g_sms[kDevices];
std::atomic<int*> g_words[kDevices];
}  // namespace

namespace sl {

Device current_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return {0, 0, nullptr};
  }
  if (dev < kDevices) {
    int* const word = g_words[dev].load(std::memory_order_acquire);
    if (word != nullptr) return {dev, g_sms[dev].load(std::memory_order_relaxed), word};
  }
  int sms = 0;
  void* word = nullptr;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      cudaGetSymbolAddress(&word, g_errors) != cudaSuccess) {
    cudaGetLastError();
    return {0, 0, nullptr};
  }
  if (dev < kDevices) {
    g_sms[dev].store(sms, std::memory_order_relaxed);
    g_words[dev].store(static_cast<int*>(word), std::memory_order_release);
  }
  return {dev, sms, static_cast<int*>(word)};
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
