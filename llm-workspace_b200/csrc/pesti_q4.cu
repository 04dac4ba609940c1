// Host side of the 4-bit vocabulary projection (include/pesti_sampler.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "../../include/pesti_sampler.h"
#include "pesti_error.h"
#include "pesti_q4.cuh"

namespace {

using namespace pesti_q4;

int refuse(const char* msg) { return pesti_set_error(PESTI_E_INVALID_ARG, msg); }

bool half_or_float(pesti_dtype d) { return d == PESTI_F32 || d == PESTI_BF16 || d == PESTI_F16; }

int esize(pesti_dtype d) { return d == PESTI_F32 ? 4 : 2; }

int check_held(int64_t V, int64_t D, int64_t group, const void* q, const void* scale) {
  if (V < 1 || V > 1 << 24) return refuse("V must be 1 to 2^24");
  if (D < 1 || D > 1 << 20) return refuse("D must be 1 to 2^20");
  if (group != 32 && group != 64 && group != 128) return refuse("group must be 32, 64 or 128");
  if (!q || !scale) return refuse("null weights or scales");
  if ((uintptr_t)q % 16) return refuse("weights are not 16-byte aligned");
  if ((uintptr_t)scale % 16) return refuse("scales are not 16-byte aligned");
  return PESTI_OK;
}

long long blocks_of(int64_t D) { return (D + BLOCK - 1) / BLOCK; }

bool overlap(const void* p, __int128 np, const void* q, __int128 nq) {
  return (__int128)(uintptr_t)p < (__int128)(uintptr_t)q + nq && (__int128)(uintptr_t)q < (__int128)(uintptr_t)p + np;
}

int need_device() {
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0)
    return pesti_set_error(PESTI_E_NO_DEVICE, "no CUDA device available");
  return PESTI_OK;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, what);
}

int check_plain(const void* w, pesti_dtype dtype, int64_t V, int64_t D, int64_t ld, int64_t group, const void* q,
                const void* scale) {
  if (!half_or_float(dtype)) return refuse("the head must be f32, bf16 or f16");
  const int rc = check_held(V, D, group, q, scale);
  if (rc) return rc;
  if (ld < D && V > 1) return refuse("ld is below D");
  if (!w) return refuse("null head");
  if ((uintptr_t)w % esize(dtype)) return refuse("the head is not aligned to its type");
  const long long n = V * blocks_of(D);
  const __int128 plain = ((__int128)(V - 1) * ld + D) * esize(dtype);
  if (overlap(w, plain, q, (__int128)n * BLOCK_BYTES) || overlap(w, plain, scale, (__int128)n * (BLOCK / group) * 2) ||
      overlap(q, (__int128)n * BLOCK_BYTES, scale, (__int128)n * (BLOCK / group) * 2))
    return refuse("head, weights and scales overlap");
  return PESTI_OK;
}

// Blocks of a row that a team of lanes takes at once.
template <typename T>
constexpr int per(bool there) {
  return there ? (sizeof(T) == 4 ? 2 : 4) : 4;
}

template <typename T, int GROUP>
int convert(bool there, const void* w, int64_t V, int64_t D, int64_t ld, void* q, void* scale, cudaStream_t st) {
  Held<T> a;
  a.w = (const T*)w;
  a.ld = ld;
  a.q = (uint32_t*)q;
  a.scale = (__nv_bfloat16*)scale;
  a.D = (int)D;
  a.blocks = (int)blocks_of(D);
  a.runs = (a.blocks + per<T>(there) - 1) / per<T>(there);
  a.total = V * a.runs;
  const int align = there || sizeof(T) == 4 ? 32 : 16, teams = there ? 32 : 16;  // of a thread block
  a.vec = (uintptr_t)w % align == 0 && (V == 1 || ld * sizeof(T) % align == 0);
  const long long grid = (a.total + teams - 1) / teams;
  if (grid > INT_MAX) return refuse("V * D too large");
  if (there)
    q4_quantize_kernel<T, GROUP, per<T>(true)><<<(unsigned)grid, 256, 0, st>>>(a);
  else
    q4_dequantize_kernel<T, GROUP, per<T>(false)><<<(unsigned)grid, 256, 0, st>>>(a);
  return launched("q4 conversion launch");
}

template <typename T>
int convert(bool there, int64_t group, const void* w, int64_t V, int64_t D, int64_t ld, void* q, void* scale,
            cudaStream_t st) {
  if (group == 32) return convert<T, 32>(there, w, V, D, ld, q, scale, st);
  if (group == 64) return convert<T, 64>(there, w, V, D, ld, q, scale, st);
  return convert<T, 128>(there, w, V, D, ld, q, scale, st);
}

int convert(bool there, pesti_dtype dtype, int64_t group, const void* w, int64_t V, int64_t D, int64_t ld, void* q,
            void* scale, cudaStream_t st) {
  if (dtype == PESTI_F32) return convert<float>(there, group, w, V, D, ld, q, scale, st);
  if (dtype == PESTI_BF16) return convert<__nv_bfloat16>(there, group, w, V, D, ld, q, scale, st);
  return convert<__half>(there, group, w, V, D, ld, q, scale, st);
}

// Column tiles of a pass over the weight, and the rows of x that fill them.
int column_tiles(int64_t columns) { return columns <= 8 ? 1 : columns <= 16 ? 2 : columns <= 32 ? 4 : 8; }

int pieces_of(pesti_dtype d) { return d == PESTI_F32 ? 3 : 1; }

long long frag_bytes(int64_t D, int tiles) { return blocks_of(D) * 4 * tiles * 32 * 16; }

template <typename T, int GROUP, int NT>
int logits_pass(LogitArgs a, cudaStream_t st) {
  q4_fragments_kernel<T, NT><<<(unsigned)a.blocks, 128, 0, st>>>(a);
  int rc = launched("q4_fragments_kernel launch");
  if (rc) return rc;
  a.k_warps = a.blocks >= 16 ? 8 : a.blocks >= 8 ? 4 : a.blocks >= 4 ? 2 : 1;
  const int rows = WARPS / a.k_warps * ROWS;
  q4_logits_kernel<std::is_same<T, __half>::value, GROUP, NT>
      <<<(unsigned)((a.V + rows - 1) / rows), WARPS * 32, 0, st>>>(a);
  return launched("q4_logits_kernel launch");
}

template <typename T, int GROUP>
int logits_tiles(const LogitArgs& a, int tiles, cudaStream_t st) {
  if (tiles == 1) return logits_pass<T, GROUP, 1>(a, st);
  if (tiles == 2) return logits_pass<T, GROUP, 2>(a, st);
  if (tiles == 4) return logits_pass<T, GROUP, 4>(a, st);
  return logits_pass<T, GROUP, 8>(a, st);
}

template <typename T>
int logits(LogitArgs a, int64_t group, int64_t B, pesti_dtype out, cudaStream_t st) {
  const char* x = (const char*)a.x;
  char* y = (char*)a.y;
  const int most = 64 / a.pieces;
  for (int64_t r = 0; r < B; r += most) {
    a.rows = (int)std::min<int64_t>(most, B - r);
    a.columns = a.rows * a.pieces;
    a.x = x + r * a.x_ld * sizeof(T);
    a.y = y + r * a.y_ld * esize(out);
    const int tiles = column_tiles(a.columns);
    const int rc = group == 32   ? logits_tiles<T, 32>(a, tiles, st)
                   : group == 64 ? logits_tiles<T, 64>(a, tiles, st)
                                 : logits_tiles<T, 128>(a, tiles, st);
    if (rc) return rc;
  }
  return PESTI_OK;
}

}  // namespace

extern "C" {

int pesti_q4_quantize(const void* d_head, pesti_dtype dtype, int64_t V, int64_t D, int64_t ld, int64_t group,
                      void* d_q, void* d_scale, void* stream) {
  int rc = check_plain(d_head, dtype, V, D, ld, group, d_q, d_scale);
  if (!rc) rc = need_device();
  return rc ? rc : convert(true, dtype, group, d_head, V, D, ld, d_q, d_scale, (cudaStream_t)stream);
}

int pesti_q4_dequantize(const void* d_q, const void* d_scale, int64_t V, int64_t D, int64_t group, void* d_head,
                        pesti_dtype dtype, int64_t ld, void* stream) {
  int rc = check_plain(d_head, dtype, V, D, ld, group, d_q, d_scale);
  if (!rc) rc = need_device();
  return rc ? rc
            : convert(false, dtype, group, d_head, V, D, ld, const_cast<void*>(d_q), const_cast<void*>(d_scale),
                      (cudaStream_t)stream);
}

int64_t pesti_q4_logits_workspace(pesti_dtype dtype, int64_t B, int64_t D) {
  if (!half_or_float(dtype)) return refuse("x must be f32, bf16 or f16");
  if (B < 0) return refuse("B < 0");
  if (B > 1 << 24) return refuse("B must be at most 2^24");
  if (D < 1 || D > 1 << 20) return refuse("D must be 1 to 2^20");
  const int p = pieces_of(dtype);
  return frag_bytes(D, column_tiles(std::min<int64_t>(B, 64 / p) * p));
}

int pesti_q4_logits(const void* d_x, pesti_dtype dtype, int64_t B, int64_t D, int64_t x_ld, const void* d_q,
                    const void* d_scale, int64_t V, int64_t group, void* d_logits, pesti_dtype out_dtype, int64_t ld,
                    void* d_ws, int64_t ws_bytes, void* stream) {
  const int64_t need = pesti_q4_logits_workspace(dtype, B, D);
  if (need < 0) return (int)need;
  int rc = check_held(V, D, group, d_q, d_scale);
  if (rc) return rc;
  if (!half_or_float(out_dtype)) return refuse("logits must be f32, bf16 or f16");
  if (B == 0) return PESTI_OK;
  if (x_ld < 0) return refuse("negative stride");  // one row may stand for all (stride 0)
  if (ld < V && B > 1) return refuse("ld is below V");
  if (!d_x || !d_logits) return refuse("null x or logits");
  if ((uintptr_t)d_x % esize(dtype)) return refuse("x is not aligned to its type");
  if ((uintptr_t)d_logits % esize(out_dtype)) return refuse("logits are not aligned to their type");
  const __int128 nx = ((__int128)(B - 1) * x_ld + D) * esize(dtype), ny = ((__int128)(B - 1) * ld + V) * esize(out_dtype);
  const __int128 nb = (__int128)V * blocks_of(D);
  if (overlap(d_logits, ny, d_x, nx) || overlap(d_logits, ny, d_q, nb * BLOCK_BYTES) ||
      overlap(d_logits, ny, d_scale, nb * (BLOCK / group) * 2))
    return refuse("inputs and logits overlap");
  if (!d_ws || ws_bytes < need) return refuse("workspace too small");
  if ((uintptr_t)d_ws % 256) return refuse("workspace is not 256-byte aligned");
  rc = need_device();
  if (rc) return rc;
  LogitArgs a = {};
  a.x = d_x;
  a.x_ld = x_ld;
  a.D = (int)D;
  a.pieces = pieces_of(dtype);
  a.q = (const uint4*)d_q;
  a.scale = (const __nv_bfloat16*)d_scale;
  a.V = (int)V;
  a.blocks = (int)blocks_of(D);
  a.frags = (uint4*)d_ws;
  a.y = d_logits;
  a.y_ld = ld;
  a.out = out_dtype == PESTI_F32 ? 0 : out_dtype == PESTI_BF16 ? 1 : 2;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PESTI_F32) return logits<float>(a, group, B, out_dtype, st);
  if (dtype == PESTI_BF16) return logits<__nv_bfloat16>(a, group, B, out_dtype, st);
  return logits<__half>(a, group, B, out_dtype, st);
}

}  // extern "C"
