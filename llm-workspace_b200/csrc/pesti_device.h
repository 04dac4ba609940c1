// The calling thread's current device, and kernels' shared memory, asked of the driver once.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/pesti_sampler.h"
#include "pesti_error.h"

constexpr int PESTI_MOST_DEVICES = 64;  // whose answers are remembered

// The device and its number of SMs.
static inline int pesti_current_device(int& device, int& sms) {
  static std::atomic<int> known[PESTI_MOST_DEVICES];
  if (cudaGetDevice(&device) != cudaSuccess) {
    (void)cudaGetLastError();
    return pesti_set_error(PESTI_E_NO_DEVICE, "no CUDA device available");
  }
  const bool remembered = device < PESTI_MOST_DEVICES;
  if (remembered && (sms = known[device].load(std::memory_order_relaxed)) > 0) return PESTI_OK;
  const cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return pesti_set_cuda_error(e, "device query");
  if (remembered) known[device].store(sms, std::memory_order_relaxed);
  return PESTI_OK;
}

// For tests (pesti_testing_give_up): the product whose sums are taken as if a wait for them had given up, and the round.
constexpr int PESTI_Q4_SUMS = 4;  // 0 to 3: the epilogues of the cross entropy's products
inline std::atomic<int64_t> pesti_give_up_at{0xffffffffLL};
static inline int pesti_give_up(int product) {
  const int64_t at = pesti_give_up_at.load(std::memory_order_relaxed);
  return at >> 32 == product ? (int)(uint32_t)at : -1;
}

// Lets `kernel` have `bytes` of dynamic shared memory on `device`; `had` is the kernel's own record of what it may have.
struct PestiShared {
  std::atomic<int> bytes[PESTI_MOST_DEVICES];
};
template <typename K>
int pesti_allow_shared(PestiShared& had, K kernel, int device, int bytes, const char* what) {
  const bool remembered = device < PESTI_MOST_DEVICES;
  if (bytes <= 48 << 10 || (remembered && had.bytes[device].load(std::memory_order_relaxed) >= bytes)) return PESTI_OK;
  int most = bytes;
  if (remembered) {  // as much as there is, so that it need not be asked again
    const cudaError_t e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
    if (e != cudaSuccess) return pesti_set_cuda_error(e, what);
    cudaFuncAttributes f;
    if (cudaFuncGetAttributes(&f, kernel) == cudaSuccess) most -= (int)f.sharedSizeBytes;
    if (most < bytes) most = bytes;
  }
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) return pesti_set_cuda_error(e, what);
  if (remembered) had.bytes[device].store(most, std::memory_order_relaxed);
  return PESTI_OK;
}
