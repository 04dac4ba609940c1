// Host side of the distillation entry points (include/pesti_sampler.h).
#include <cuda_runtime.h>

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
  if (V < 1 || V > 0x7fffffffLL) return refuse("V must be 1 to 2^31-1");
  if (ld < V) return refuse("ld is below V");
  if (k < 1 || k > PESTI_DISTILL_MAX_TOP) return refuse("k must be 1 to 256");
  // one value may stand for all rows (stride 0)
  if (idx_ld < 0 || val_ld < 0) return refuse("negative stride");
  if (!(temperature >= 0x1p-10 && temperature <= 0x1p20)) return refuse("temperature must be 2^-10 to 2^20");
  if (N == 0) return PESTI_OK;
  if (!d_logits || !d_idx || !d_val) return refuse("null logits or teacher list");
  if ((uintptr_t)d_logits % esize(dtype)) return refuse("logits are not aligned to their type");
  if ((uintptr_t)d_val % esize(val_dtype)) return refuse("teacher values are not aligned to their type");
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
  // below C, so that c_lo > 0 and -inf stays -inf in x*c + x*c_lo (with c_lo = 0, as T = 1/ln 2 would have it, NaN)
  a.c = (float)a.C;
  if ((double)a.c >= a.C) a.c = std::nextafter(a.c, 0.0f);
  a.c_lo = (float)(a.C - (double)a.c);
  a.units = dtype == PESTI_F32 ? row_units<float>(V) : row_units<__half>(V);
  return PESTI_OK;
}

int need_device() {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0)
    return pesti_set_error(PESTI_E_NO_DEVICE, "no CUDA device available");
  return PESTI_OK;
}

long long up256(long long n) { return (n + 255) / 256 * 256; }

// Lays the scratch out behind `base` (which may be null, for the size alone).
long long layout(char* base, DistillArgs& a, long long N, long long units, int k) {
  const long long parts = up256(N * units * (long long)sizeof(Partial));
  const long long lists = up256(N * lists_of(k) * (long long)sizeof(double));
  a.parts = (Partial*)base;
  a.lists = (double*)(base + parts);
  a.stats = (double*)(base + parts + lists);
  return parts + lists + up256(N * stats_of(k) * (long long)sizeof(double));
}

// A launch that may start before its predecessor has ended (and waits for it).
template <typename... K, typename... A>
int launch_behind(const char* what, void (*kernel)(K...), long long blocks, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, K(args)...);
  return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, what);
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, what);
}

template <typename T>
int run(const DistillArgs& a, cudaStream_t st) {
  const long long per_row = (a.units + UNIT_WARPS - 1) / UNIT_WARPS, lists = (a.N + UNIT_WARPS - 1) / UNIT_WARPS;
  if (a.N > (0x7fffffffLL - lists) / per_row) return refuse("N * V too large");
  distill_scan_kernel<T><<<(unsigned)(lists + a.N * per_row), UNIT_WARPS * 32, 0, st>>>(a, lists, per_row);
  int rc = launched("distill_scan_kernel launch");
  if (rc) return rc;
  rc = launch_behind("distill_join_kernel launch", distill_join_kernel<T>, (a.N + JOIN_WARPS - 1) / JOIN_WARPS,
                     JOIN_WARPS * 32, st, a);
  if (rc || !a.grad) return rc;
  return launch_behind("distill_backward_kernel launch", distill_backward_kernel<T>, a.N * per_row, UNIT_WARPS * 32, st,
                       a, per_row);
}

template <typename T>
int launch_backward(const DistillArgs& a, long long N, cudaStream_t st) {
  const long long per_row = (a.units + UNIT_WARPS - 1) / UNIT_WARPS;
  if (N > 0x7fffffffLL / per_row) return refuse("N * V too large");
  distill_backward_kernel<T><<<(unsigned)(N * per_row), UNIT_WARPS * 32, 0, st>>>(a, per_row);
  return launched("distill_backward_kernel launch");
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

int64_t pesti_distill_topk_workspace(pesti_dtype dtype, int64_t N, int64_t V, int64_t k) {
  if (!half_or_float(dtype)) return refuse("logits must be f32, bf16 or f16");
  if (N < 0) return refuse("N < 0");
  if (V < 1 || V > 0x7fffffffLL) return refuse("V must be 1 to 2^31-1");
  if (k < 1 || k > PESTI_DISTILL_MAX_TOP) return refuse("k must be 1 to 256");
  const long long units = dtype == PESTI_F32 ? row_units<float>(V) : row_units<__half>(V);
  if (N > 0x7fffffffLL / units) return refuse("N * V too large");
  DistillArgs a;
  return layout(nullptr, a, N, units, (int)k);
}

int pesti_distill_topk(const void* d_logits, pesti_dtype dtype, int64_t N, int64_t V, int64_t ld,
                       const int32_t* d_idx, int64_t idx_ld, const void* d_val, pesti_dtype val_dtype,
                       int64_t val_ld, int64_t k, const float* d_teacher_lse, const float* d_weight,
                       double temperature, float* d_loss, double* d_stats, void* d_grad, int64_t grad_ld,
                       void* d_ws, int64_t ws_bytes, void* stream) {
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
  if (N > 0x7fffffffLL / a.units) return refuse("N * V too large");
  const long long need = layout((char*)d_ws, a, N, a.units, a.k);
  if (!d_ws || ws_bytes < need) return refuse("workspace too small");
  if ((uintptr_t)d_ws % 256) return refuse("workspace is not 256-byte aligned");
  a.loss = d_loss;
  if (d_stats)
    a.stats = d_stats;
  else if (!d_grad)
    a.stats = nullptr;
  a.grad = d_grad;
  a.grad_ld = grad_ld;
  a.N = N;
  rc = need_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PESTI_F32) return run<float>(a, st);
  if (dtype == PESTI_BF16) return run<__nv_bfloat16>(a, st);
  return run<__half>(a, st);
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
  a.N = N;
  rc = need_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PESTI_F32) return launch_backward<float>(a, N, st);
  if (dtype == PESTI_BF16) return launch_backward<__nv_bfloat16>(a, N, st);
  return launch_backward<__half>(a, N, st);
}

}  // extern "C"
