// Host side of the 4-bit vocabulary projection (include/pesti_sampler.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "../../include/pesti_sampler.h"
#include "pesti_device.h"
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

// Tiles of the held weight; its bytes are TILE_BYTES of q a tile, and ROWS * BLOCK / group scales.
long long tiles_of(int64_t V, int64_t D) { return (V + ROWS - 1) / ROWS * blocks_of(D); }

constexpr int TILE_BYTES = TILE_WORDS * 4;

bool overlap(const void* p, __int128 np, const void* q, __int128 nq) {
  return (__int128)(uintptr_t)p < (__int128)(uintptr_t)q + nq && (__int128)(uintptr_t)q < (__int128)(uintptr_t)p + np;
}

struct Device {
  int index, sms;
};

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
  const __int128 tiles = tiles_of(V, D), held = tiles * TILE_BYTES, scales = tiles * (ROWS * BLOCK / group) * 2;
  const __int128 plain = ((__int128)(V - 1) * ld + D) * esize(dtype);
  if (overlap(w, plain, q, held) || overlap(w, plain, scale, scales) || overlap(q, held, scale, scales))
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
  a.V = (int)V;
  a.runs = (a.blocks + per<T>(there) - 1) / per<T>(there);
  a.total = (V + ROWS - 1) / ROWS * (there ? ROWS : ROWS / 16) * a.runs;
  const int align = there || sizeof(T) == 4 ? 32 : 16, runs = there ? 32 : 1;  // of a thread block
  a.vec = (uintptr_t)w % align == 0 && (V == 1 || ld * sizeof(T) % align == 0);
  const long long grid = (a.total + runs - 1) / runs;
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

constexpr int MOST_ROWS = 64;            // of x, a pass over the weight
constexpr int SHARED_BYTES = 200 << 10;  // for the stages
constexpr int FEW_BYTES = 196 << 10;     // for few rows of x, beside 30 KB of sums

int pieces_of(pesti_dtype d) { return d == PESTI_F32 ? pieces<float> : 1; }

int columns_of(int64_t rows) { return (int)(rows + 15) / 16 * 16; }

// Few rows of x that fit shared memory whole.  A column tile of the products by warps holds 8; f32 rows cost them two
// products, and each row some us before the first, so that more than 4 pay from 2048 columns on (us for 5 / 8, and on
// tensor memory: 128256 x 4096: 78 / 82, 92 / 93; 8000 x 4096: 14 / 17, 22; 32000 x 2048: 18 / 20, 18 / 19; 32001 x 1000:
// 12 / 14, 11 / 12).
bool few(int64_t D, int pieces, int64_t rows) {
  return rows <= (pieces == 1 || D >= 2048 ? 8 : 4) && blocks_of(D) * rows * pieces * (BLOCK * 2) <= FEW_BYTES;
}

// How a pass with few rows shares its tiles and their K out: the least time of the busiest SM, by the weight's bytes that it
// reads (44 bytes a nanosecond), half a microsecond per round of tiles, and 50 ns for each part of a sum that is joined.
int k_warps_of(long long stacks, int blocks, int warps, int sms) {
  double best = 1e30;
  int at = 1;
  for (int kw = 1; kw <= warps && kw <= blocks; ++kw) {
    if (warps % kw || (kw > 1 && warps / kw > MOST_SLOTS)) continue;
    const int slots = warps / kw, turns = (blocks + kw - 1) / kw;
    const long long rounds = (stacks + (long long)sms * slots - 1) / ((long long)sms * slots);
    const double t = (double)rounds * (warps * turns * TILE_BYTES / 44.0 + 500.0 + 50.0 * kw);
    if (t < best) {
      best = t;
      at = kw;
    }
  }
  return at;
}

template <typename... K, typename... A>
int launch(const char* what, void (*kernel)(K...), long long blocks, int threads, int smem, cudaStream_t st,
           const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, K(args)...);
  return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, what);
}

template <int P, int GROUP, int COLUMNS>
int wide_pass(const LogitArgs& a, Device dev, cudaStream_t st) {
  const auto kernel = q4_wide_kernel<P, GROUP, COLUMNS>;
  const int smem = 1024 + a.stages * (SLOTS * WIDE_BYTES + COLUMNS * P * (BLOCK * 2));
  static PestiShared shared;
  const int rc = pesti_allow_shared(shared, kernel, dev.index, smem, "q4_wide_kernel shared memory");
  if (rc) return rc;
  return launch("q4_wide_kernel launch", kernel, std::min(dev.sms, a.stacks), WIDE_THREADS, smem, st, a);
}

template <typename T, int GROUP>
int pass(LogitArgs a, Device dev, cudaStream_t st) {
  constexpr int P = pieces<T>;
  if (few(a.D, P, a.rows)) {
    a.stacks = (a.V + ROWS - 1) / ROWS;
    a.k_warps = k_warps_of(a.stacks, a.blocks, FEW_WARPS, dev.sms);
    const int slots = FEW_WARPS / a.k_warps;
    const int smem = a.blocks * a.rows * P * (BLOCK * 2) + 16 + (FEW_WARPS - slots) * 16 * 32 * 4;
    const auto kernel = q4_logits_kernel<T, GROUP>;
    static PestiShared shared;
    const int rc = pesti_allow_shared(shared, kernel, dev.index, smem, "q4_logits_kernel shared memory");
    if (rc) return rc;
    return launch("q4_logits_kernel launch", kernel, std::min<long long>(dev.sms, (a.stacks + slots - 1) / slots),
                  FEW_WARPS * 32, smem, st, a);
  }
  a.stacks = (a.V + WIDE - 1) / WIDE;
  const int columns = columns_of(a.rows);
  const int rc = launch("q4_operand_kernel launch", q4_operand_kernel<T>, columns, 256, 0, st, a, columns);
  if (rc) return rc;
  a.give_up = pesti_give_up(PESTI_Q4_SUMS);
  a.stages = std::min(8, SHARED_BYTES / (SLOTS * WIDE_BYTES + columns * P * (BLOCK * 2)));
  if (columns == 16) return wide_pass<P, GROUP, 16>(a, dev, st);
  if (columns == 32) return wide_pass<P, GROUP, 32>(a, dev, st);
  if (columns == 48) return wide_pass<P, GROUP, 48>(a, dev, st);
  return wide_pass<P, GROUP, 64>(a, dev, st);
}

template <typename T>
int logits(LogitArgs a, int64_t group, int64_t B, pesti_dtype out, Device dev, cudaStream_t st) {
  const char* x = (const char*)a.x;
  char* y = (char*)a.y;
  for (int64_t r = 0; r < B; r += MOST_ROWS) {
    a.rows = (int)std::min<int64_t>(MOST_ROWS, B - r);
    a.x = x + r * a.x_ld * sizeof(T);
    a.x_vec = (uintptr_t)a.x % 16 == 0 && a.x_ld * sizeof(T) % 16 == 0;
    a.y = y + r * a.y_ld * esize(out);
    const int rc = group == 32   ? pass<T, 32>(a, dev, st)
                   : group == 64 ? pass<T, 64>(a, dev, st)
                                 : pass<T, 128>(a, dev, st);
    if (rc) return rc;
  }
  return PESTI_OK;
}

}  // namespace

extern "C" {

int pesti_q4_quantize(const void* d_head, pesti_dtype dtype, int64_t V, int64_t D, int64_t ld, int64_t group,
                      void* d_q, void* d_scale, void* stream) {
  int rc = check_plain(d_head, dtype, V, D, ld, group, d_q, d_scale);
  Device dev = {};
  if (!rc) rc = pesti_current_device(dev.index, dev.sms);
  return rc ? rc : convert(true, dtype, group, d_head, V, D, ld, d_q, d_scale, (cudaStream_t)stream);
}

int pesti_q4_dequantize(const void* d_q, const void* d_scale, int64_t V, int64_t D, int64_t group, void* d_head,
                        pesti_dtype dtype, int64_t ld, void* stream) {
  int rc = check_plain(d_head, dtype, V, D, ld, group, d_q, d_scale);
  Device dev = {};
  if (!rc) rc = pesti_current_device(dev.index, dev.sms);
  return rc ? rc
            : convert(false, dtype, group, d_head, V, D, ld, const_cast<void*>(d_q), const_cast<void*>(d_scale),
                      (cudaStream_t)stream);
}

int64_t pesti_q4_logits_workspace(pesti_dtype dtype, int64_t B, int64_t D) {
  if (!half_or_float(dtype)) return refuse("x must be f32, bf16 or f16");
  if (B < 0) return refuse("B < 0");
  if (B > 1 << 24) return refuse("B must be at most 2^24");
  if (D < 1 || D > 1 << 20) return refuse("D must be 1 to 2^20");
  if (few(D, pieces_of(dtype), B)) return 0;
  // the operand, and each row's power of two
  const int64_t columns = columns_of(std::min<int64_t>(B, MOST_ROWS));
  return columns * (blocks_of(D) * pieces_of(dtype) * (BLOCK * 2) + 8);
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
  const __int128 tiles = tiles_of(V, D);
  if (overlap(d_logits, ny, d_x, nx) || overlap(d_logits, ny, d_q, tiles * TILE_BYTES) ||
      overlap(d_logits, ny, d_scale, tiles * (ROWS * BLOCK / group) * 2))
    return refuse("inputs and logits overlap");
  if (need && (!d_ws || ws_bytes < need)) return refuse("workspace too small");
  if ((uintptr_t)d_ws % 256) return refuse("workspace is not 256-byte aligned");
  Device dev = {};
  rc = pesti_current_device(dev.index, dev.sms);
  if (rc) return rc;
  LogitArgs a = {};
  a.x = d_x;
  a.x_ld = x_ld;
  a.D = (int)D;
  a.q = (const uint4*)d_q;
  a.scale = (const __nv_bfloat16*)d_scale;
  a.V = (int)V;
  a.blocks = (int)blocks_of(D);
  a.operand = (uint4*)d_ws;
  a.y = d_logits;
  a.y_ld = ld;
  a.out = out_dtype == PESTI_F32 ? 0 : out_dtype == PESTI_BF16 ? 1 : 2;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PESTI_F32) return logits<float>(a, group, B, out_dtype, dev, st);
  if (dtype == PESTI_BF16) return logits<__nv_bfloat16>(a, group, B, out_dtype, dev, st);
  return logits<__half>(a, group, B, out_dtype, dev, st);
}

}  // extern "C"
