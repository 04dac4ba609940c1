// Host side of the distillation entry points (include/pesti_sampler.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "../../include/pesti_sampler.h"
#include "pesti_distill.cuh"
#include "pesti_error.h"

namespace {

using namespace pesti_rows;

int refuse(const char* msg) { return pesti_set_error(PESTI_E_INVALID_ARG, msg); }

bool half_or_float(pesti_dtype d) { return d == PESTI_F32 || d == PESTI_BF16 || d == PESTI_F16; }

int esize(pesti_dtype d) { return d == PESTI_F32 ? 4 : 2; }

// The checks both calls share; fills the arguments that do not depend on the call.
int common(DistillArgs& a, const void* d_logits, pesti_dtype dtype, int64_t N, int64_t V, int64_t ld,
           const int32_t* d_idx, int64_t idx_ld, const void* d_val, pesti_dtype val_dtype, int64_t val_ld, int64_t k,
           const float* d_teacher_lse, const float* d_weight, double temperature) {
  if (!half_or_float(dtype)) return refuse("logits must be f32, bf16 or f16");
  if (!half_or_float(val_dtype)) return refuse("teacher values must be f32, bf16 or f16");
  if (N < 0) return refuse("N < 0");
  if (N > 0x7fffffffLL) return refuse("N must be below 2^31");
  if (V < 1 || V > (1LL << 30)) return refuse("V must be 1 to 2^30");
  if (ld < V) return refuse("ld is below V");
  if (k < 1 || k > PESTI_DISTILL_MAX_TOP) return refuse("k must be 1 to 256");
  // one value may stand for all rows (stride 0)
  if (idx_ld < 0 || val_ld < 0) return refuse("negative stride");
  if (!(temperature >= 0x1p-10 && temperature <= 0x1p20)) return refuse("temperature must be 2^-10 to 2^20");
  if (N == 0) return PESTI_OK;
  if (!d_logits || !d_idx || !d_val) return refuse("null logits or teacher list");
  if ((uintptr_t)d_logits % esize(dtype)) return refuse("logits are not aligned to their type");
  a = DistillArgs{};
  a.logits = d_logits;
  a.ld = ld;
  a.V = V;
  a.idx = d_idx;
  a.val = d_val;
  a.idx_ld = idx_ld;
  a.val_ld = val_ld;
  a.val_dtype = val_dtype == PESTI_F32 ? 0 : val_dtype == PESTI_BF16 ? 1 : 2;
  a.k = (int)k;
  a.teacher_lse = d_teacher_lse;
  a.weight = d_weight;
  a.T = temperature;
  a.C = 1.4426950408889634074 / a.T;
  // rounded down, so that c_lo >= 0 and -inf stays -inf in x*c + x*c_lo
  a.c = (float)a.C;
  if ((double)a.c > a.C) a.c = std::nextafter(a.c, 0.0f);
  a.c_lo = (float)(a.C - (double)a.c);
  a.units = dtype == PESTI_F32 ? row_units<float>(V) : row_units<__half>(V);
  return PESTI_OK;
}

struct Device {
  std::atomic<int> sms{0};  // 0: not set up yet
};
constexpr int kMaxDevices = 64;
Device g_devices[kMaxDevices];

constexpr int kMaxSlots = 3;

template <typename T, bool GRAD>
cudaError_t allow() {
  cudaError_t e = cudaFuncSetAttribute(distill_row_kernel<T, GRAD>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(distill_row_kernel<T, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              ROW_WARPS * MAX_KEEP * 512);
}

int set_up(int* sms) {
  int n = 0, dev = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0)
    return pesti_set_error(PESTI_E_NO_DEVICE, "no CUDA device available");
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return pesti_set_cuda_error(e, "cudaGetDevice");
  if (dev >= kMaxDevices) return refuse("device index out of range");
  int have = g_devices[dev].sms.load(std::memory_order_acquire);
  if (have == 0) {
    e = cudaDeviceGetAttribute(&have, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = allow<float, false>();
    if (e == cudaSuccess) e = allow<float, true>();
    if (e == cudaSuccess) e = allow<__nv_bfloat16, false>();
    if (e == cudaSuccess) e = allow<__nv_bfloat16, true>();
    if (e == cudaSuccess) e = allow<__half, false>();
    if (e == cudaSuccess) e = allow<__half, true>();
    if (e != cudaSuccess) return pesti_set_cuda_error(e, "distillation kernels' set-up");
    g_devices[dev].sms.store(have, std::memory_order_release);
  }
  *sms = have;
  return PESTI_OK;
}

// A warp's part of a row that is split over c CTAs, and its batches.
template <typename T>
void split(DistillArgs& a, long long c) {
  const long long seg = 512 / (long long)sizeof(T), ve = 16 / (long long)sizeof(T);
  const long long segs = (a.V + ve - 1 + seg - 1) / seg;
  a.warp_segs = (int)((segs + c * ROW_WARPS - 1) / (c * ROW_WARPS));
  a.batches = (a.warp_segs + BATCH - 1) / BATCH;
}

template <typename T, bool GRAD>
int launch_row(DistillArgs& a, long long N, int sms, cudaStream_t st) {
  // The cluster: as many CTAs as keep a row in shared memory, more while the
  // rows alone do not fill the GPU and every warp still has a segment.  Without
  // a gradient nothing stays, and the split only evens out the last round.
  long long c = 1;
  split<T>(a, c);
  a.keep = 0;
  if (GRAD) {
    while (c < MAX_CLUSTER && a.warp_segs > MAX_KEEP) split<T>(a, c *= 2);
    a.keep = a.warp_segs <= MAX_KEEP;
    if (!a.keep) split<T>(a, c = 1);
  } else {
    const long long all = 2LL * sms;
    auto share = [&](long long k) { return (double)N / (double)((N * k + all - 1) / all) * (double)k / (double)all; };
    while (c < 4 && N * c > all && share(c) < 0.93) c *= 2;
  }
  while (c < MAX_CLUSTER && N * c < sms && a.warp_segs > 1) split<T>(a, c *= 2);
  split<T>(a, c);
  a.slots = a.keep ? a.batches : std::min(kMaxSlots, GRAD ? 2 * a.batches : a.batches);
  a.ring_segs = std::min(a.warp_segs, a.slots * BATCH);
  a.N = N;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(ROW_THREADS);
  cfg.dynamicSmemBytes = (size_t)ROW_WARPS * a.ring_segs * 512;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // as many clusters as run at once (clusters of more than two CTAs may leave SMs of a GPC over)
  long long clusters = N;
  if (N * c > sms) {
    cfg.gridDim = dim3((unsigned)c);
    int most = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&most, distill_row_kernel<T, GRAD>, &cfg);
    if (e != cudaSuccess) return pesti_set_cuda_error(e, "cudaOccupancyMaxActiveClusters");
    if (most < 1) return refuse("no room for a cluster");
    clusters = std::min<long long>(N, most);
  }
  cfg.gridDim = dim3((unsigned)(clusters * c));
  const cudaError_t e = cudaLaunchKernelEx(&cfg, distill_row_kernel<T, GRAD>, (const DistillArgs)a);
  return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, "distill_row_kernel launch");
}

template <typename T>
int launch_backward(const DistillArgs& a, long long N, cudaStream_t st) {
  const long long per_row = (a.units + BACK_WARPS - 1) / BACK_WARPS;
  if (N > 0x7fffffffLL / per_row) return refuse("N * V too large");
  distill_backward_kernel<T><<<(unsigned)(N * per_row), BACK_WARPS * 32, 0, st>>>(a, per_row);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, "distill_backward_kernel launch");
}

int check_grad(const void* d_logits, pesti_dtype dtype, int64_t N, int64_t V, int64_t ld, const void* d_grad,
               int64_t grad_ld) {
  if (grad_ld < V) return refuse("grad_ld is below V");
  if ((uintptr_t)d_grad % esize(dtype)) return refuse("gradient is not aligned to its type");
  if (d_grad == d_logits) return grad_ld == ld ? PESTI_OK : refuse("a gradient in place needs grad_ld == ld");
  const char *p = (const char*)d_logits, *q = (const char*)d_grad;
  const __int128 np = ((__int128)(N - 1) * ld + V) * esize(dtype), nq = ((__int128)(N - 1) * grad_ld + V) * esize(dtype);
  if (np > LLONG_MAX || nq > LLONG_MAX) return refuse("N * ld too large");
  if (p < q + (long long)nq && q < p + (long long)np) return refuse("logits and gradient overlap");
  return PESTI_OK;
}

}  // namespace

extern "C" {

int pesti_distill_topk(const void* d_logits, pesti_dtype dtype, int64_t N, int64_t V, int64_t ld,
                       const int32_t* d_idx, int64_t idx_ld, const void* d_val, pesti_dtype val_dtype,
                       int64_t val_ld, int64_t k, const float* d_teacher_lse, const float* d_weight,
                       double temperature, float* d_loss, double* d_stats, void* d_grad, int64_t grad_ld,
                       void* stream) {
  DistillArgs a;
  int rc = common(a, d_logits, dtype, N, V, ld, d_idx, idx_ld, d_val, val_dtype, val_ld, k, d_teacher_lse, d_weight,
                  temperature);
  if (rc) return rc;
  if (N == 0) return PESTI_OK;
  if (!d_loss) return refuse("null loss");
  if (d_grad) {
    rc = check_grad(d_logits, dtype, N, V, ld, d_grad, grad_ld);
    if (rc) return rc;
    if (d_stats && d_grad == d_logits) return refuse("the backward call needs the logits: no stats with a gradient in place");
  }
  a.loss = d_loss;
  a.stats = d_stats;
  a.grad = d_grad;
  a.grad_ld = grad_ld;
  int sms = 0;
  rc = set_up(&sms);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PESTI_F32)
    return d_grad ? launch_row<float, true>(a, N, sms, st) : launch_row<float, false>(a, N, sms, st);
  if (dtype == PESTI_BF16)
    return d_grad ? launch_row<__nv_bfloat16, true>(a, N, sms, st) : launch_row<__nv_bfloat16, false>(a, N, sms, st);
  return d_grad ? launch_row<__half, true>(a, N, sms, st) : launch_row<__half, false>(a, N, sms, st);
}

int pesti_distill_topk_backward(const void* d_logits, pesti_dtype dtype, int64_t N, int64_t V, int64_t ld,
                                const int32_t* d_idx, int64_t idx_ld, const void* d_val, pesti_dtype val_dtype,
                                int64_t val_ld, int64_t k, const float* d_teacher_lse, const float* d_weight,
                                double temperature, const double* d_stats, const float* d_up, int64_t up_stride,
                                void* d_grad, int64_t grad_ld, void* stream) {
  DistillArgs a;
  int rc = common(a, d_logits, dtype, N, V, ld, d_idx, idx_ld, d_val, val_dtype, val_ld, k, d_teacher_lse, d_weight,
                  temperature);
  if (rc) return rc;
  if (up_stride < 0) return refuse("negative stride");
  if (N == 0) return PESTI_OK;
  if (!d_stats || !d_up || !d_grad) return refuse("null stats, upstream gradient or gradient");
  rc = check_grad(d_logits, dtype, N, V, ld, d_grad, grad_ld);
  if (rc) return rc;
  a.stats = const_cast<double*>(d_stats);
  a.up = d_up;
  a.up_stride = up_stride;
  a.grad = d_grad;
  a.grad_ld = grad_ld;
  int sms = 0;
  rc = set_up(&sms);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PESTI_F32) return launch_backward<float>(a, N, st);
  if (dtype == PESTI_BF16) return launch_backward<__nv_bfloat16>(a, N, st);
  return launch_backward<__half>(a, N, st);
}

}  // extern "C"
