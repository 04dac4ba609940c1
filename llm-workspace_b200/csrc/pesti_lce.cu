// Host side of the cross entropy from hidden states (include/pesti_sampler.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "../../include/pesti_sampler.h"
#include "../../include/pesti_testing.h"
#include "pesti_device.h"
#include "pesti_error.h"
#include "pesti_lce.cuh"
#include "pesti_tensor_map.h"

namespace {

using namespace pesti_lce;

int refuse(const char* msg) { return pesti_set_error(PESTI_E_INVALID_ARG, msg); }

long long up_to(long long n, long long to) { return (n + to - 1) / to * to; }

struct Call {
  const void* hidden;
  pesti_dtype dtype;
  int64_t N, D, h_ld;
  const void* head;
  int64_t V, w_ld;
  const void* target;
  int target_bytes;
  const float* weight;
  double eps, zeta;
};

int check_sizes(pesti_dtype dtype, int64_t N, int64_t V, int64_t D) {
  if (dtype != PESTI_BF16 && dtype != PESTI_F16) return refuse("hidden states and head must be bf16 or f16");
  if (N < 0) return refuse("N < 0");
  if (N > 1 << 24) return refuse("N must be at most 2^24");
  if (V < 1 || V > 1 << 24) return refuse("V must be 1 to 2^24");
  if (D < 1 || D > 1 << 20) return refuse("D must be 1 to 2^20");
  if (up_to(N, 256) / 128 * (up_to(V, BN) / BN) > 0x3fffffff) return refuse("N * V too large");
  if (up_to(V, BN) / 128 * (up_to(D, BN) / BN) > 0x3fffffff) return refuse("V * D too large");
  if (up_to(N, 256) / 128 * (up_to(D, BN) / BN) > 0xffffff) return refuse("N * D too large");
  return PESTI_OK;
}

int check(const Call& c) {
  const int rc = check_sizes(c.dtype, c.N, c.V, c.D);
  if (rc) return rc;
  if (c.h_ld < 0) return refuse("negative stride");  // one row may stand for all (stride 0)
  if (c.w_ld < c.D) return refuse("w_ld is below D");
  if (c.w_ld % 8 || c.w_ld > 1LL << 36) return refuse("w_ld must be a multiple of 8");
  if (c.target_bytes != 4 && c.target_bytes != 8) return refuse("targets must be of 4 or 8 bytes");
  if (!(c.eps >= 0.0 && c.eps < 1.0)) return refuse("label_smoothing must be 0 to below 1");
  if (!(c.zeta >= 0.0 && c.zeta <= 1e6)) return refuse("z_loss must be 0 to 1e6");
  if (c.N == 0) return PESTI_OK;
  if (!c.hidden || !c.head || !c.target) return refuse("null hidden states, head or targets");
  if ((uintptr_t)c.hidden % 2) return refuse("hidden states are not aligned to their type");
  if ((uintptr_t)c.head % 16) return refuse("head is not 16-byte aligned");
  if ((uintptr_t)c.target % c.target_bytes) return refuse("targets are not aligned to their type");
  if ((uintptr_t)c.weight % 4) return refuse("weights are not aligned to their type");
  return PESTI_OK;
}

bool overlap(const void* p, __int128 np, const void* q, __int128 nq) {
  return (__int128)(uintptr_t)p < (__int128)(uintptr_t)q + nq && (__int128)(uintptr_t)q < (__int128)(uintptr_t)p + np;
}

int check_grads(const Call& c, const void* dh, int64_t dh_ld, const void* dw, int64_t dw_ld) {
  const __int128 h = ((__int128)(c.N - 1) * c.h_ld + c.D) * 2, w = ((__int128)(c.V - 1) * c.w_ld + c.D) * 2;
  const __int128 oh = ((__int128)(c.N - 1) * dh_ld + c.D) * 2, ow = ((__int128)(c.V - 1) * dw_ld + c.D) * 2;
  if (dh) {
    if (dh_ld < c.D && c.N > 1) return refuse("dh_ld is below D");
    if ((uintptr_t)dh % 2) return refuse("the hidden states' gradient is not aligned to its type");
    if (overlap(dh, oh, c.hidden, h) || overlap(dh, oh, c.head, w)) return refuse("inputs and gradients overlap");
  }
  if (dw) {
    if (dw_ld < c.D) return refuse("dw_ld is below D");
    if (dw_ld % 8 || dw_ld > 1LL << 36) return refuse("dw_ld must be a multiple of 8");
    if ((uintptr_t)dw % 16) return refuse("the head's gradient is not 16-byte aligned");
    if (overlap(dw, ow, c.hidden, h) || overlap(dw, ow, c.head, w)) return refuse("inputs and gradients overlap");
    if (dh && overlap(dh, oh, dw, ow)) return refuse("gradients overlap");
  }
  return PESTI_OK;
}

// How the gradients' work is cut: pieces of the vocabulary whose G stays below about 256 MB; the hidden states'
// gradient sums ranges of a piece's K in parts of their own, up to 512 MB of them.
struct Cut {
  long long piece, part_room;
};

Cut cut_of(int64_t N, int64_t V, int64_t D) {
  Cut c;
  const long long rows = std::max<long long>(256, up_to(N, 256));
  const long long most = std::max<long long>(8192, (256LL << 20) / (2 * rows));
  const long long pieces = (V + most - 1) / most;
  c.piece = up_to((V + pieces - 1) / pieces, BN);
  c.part_room = std::max(rows, std::min(64 * rows, (512LL << 20) / (4 * up_to(D, 4)) / 256 * 256));
  return c;
}

constexpr int SMS = 148;  // by which sizes of scratch are chosen

// Pairs of blocks read each operand's tile half as often, which is what large products need (4096 x 128256 x 4096: 12.7
// ms against 14.7 with single blocks); up to 128 rows the products are bound by reading the head, and a pair's second
// block would only add empty rows (16 x 152064 x 2048: 142 us against 122).
int blocks_per_tile(int64_t N) { return N > 128 ? 2 : 1; }

// Columns of the logits' tiles: 256, or fewer where that makes a twentieth fewer columns in whole rounds of tiles over
// the SMs, with 24 for a tile's own beginning and end.  (594 tiles of 256 columns are five rounds of 148, and so are 732
// of 208: 16 x 152064 x 2048 125 -> 121 us; 240 instead of 256 for 1024 x 256000 x 2048 saves a fiftieth of the columns
// and takes that much longer.)
int tile_width(int64_t N, int64_t V) {
  const int cg = blocks_per_tile(N), units = SMS / cg;
  const long long rows = (N + 128 * cg - 1) / (128 * cg);
  long long best = 0;
  int at = BN;
  for (int w = BN; w >= 128; w -= 16) {
    const long long rounds = (rows * ((V + w - 1) / w) + units - 1) / units, t = rounds * (w + 24) * (w < BN ? 20 : 19);
    if (!best || t < best) {
      best = t;
      at = w;
    }
  }
  return at;
}

struct Layout {
  Plan* plan;
  int *idx, *packed, *place;
  RowCoef* coef;
  float* zt;
  uint16_t* rows;
  float2* parts;
  float* zsum;
  uint16_t* grad;
  float* part32;
  long long rows_pad, ldc, ld32;
  int width;
  Cut cut;
  long long bytes;
};

// `forward`: with the tiles' statistics; `grads`: with a piece of G and the parts of the hidden states' gradient.
Layout layout(char* base, int64_t N, int64_t V, int64_t D, bool forward, bool grads) {
  Layout l = {};
  long long at = 0;
  auto take = [&](long long bytes) {
    char* p = base + at;
    at += up_to(bytes, 1024);
    return p;
  };
  l.rows_pad = up_to(N, 256);
  l.ldc = up_to(D, 64);  // whole lines of L2
  l.ld32 = up_to(D, 4);
  l.plan = (Plan*)take(sizeof(Plan));
  l.idx = (int*)take(l.rows_pad * 4);
  l.packed = (int*)take(l.rows_pad * 4);
  l.place = (int*)take(l.rows_pad * 4);
  l.coef = (RowCoef*)take(l.rows_pad * sizeof(RowCoef));
  l.zt = (float*)take(l.rows_pad * 4);
  l.rows = (uint16_t*)take(l.rows_pad * l.ldc * 2);
  l.width = tile_width(N, V);
  const long long tiles = (V + l.width - 1) / l.width;
  if (forward) {
    l.parts = (float2*)take(tiles * l.rows_pad * 8);
    l.zsum = (float*)take(tiles * l.rows_pad * 4);
  }
  if (grads) {
    l.cut = cut_of(N, V, D);
    l.grad = (uint16_t*)take(l.rows_pad * l.cut.piece * 2);
    l.part32 = (float*)take(l.cut.part_room * l.ld32 * 4);
  }
  l.bytes = at;
  return l;
}

struct Device {
  int index, sms;
};

// Every kernel waits on the device for the one before it, so it may be launched while that one still runs.
template <typename... K, typename... A>
int launch(const char* what, void (*kernel)(K...), int cg, dim3 blocks, int threads, int smem, cudaStream_t st,
           const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cg;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cg > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, K(args)...);
  return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, what);
}

template <int CG, bool BF16, bool A_MN, bool B_MN, Epilogue E>
int launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out, const GemmArgs& g, Device dev,
                cudaStream_t st) {
  auto kernel = head_gemm_kernel<CG, BF16, A_MN, B_MN, E>;
  static PestiShared shared;
  const int rc = pesti_allow_shared(shared, kernel, dev.index, smem_bytes(CG, E), "head_gemm_kernel shared memory");
  if (rc) return rc;
  GemmArgs args = g;
  args.give_up = pesti_give_up(E);
  return launch("head_gemm_kernel launch", kernel, CG, dim3(dev.sms / CG * CG), THREADS, smem_bytes(CG, E), st, a, b, out,
                args);
}

RowArgs row_args(const Call& c, const Layout& l, int cg, int sms) {
  RowArgs r = {};
  r.plan = l.plan;
  r.hidden = c.hidden;
  r.N = c.N;
  r.D = c.D;
  r.h_ld = c.h_ld;
  r.V = c.V;
  r.target = c.target;
  r.target_bytes = c.target_bytes;
  r.weight = c.weight;
  r.eps = (float)c.eps;
  r.zeta = (float)c.zeta;
  r.idx = l.idx;
  r.packed = l.packed;
  r.place = l.place;
  r.coef = l.coef;
  r.zt = l.zt;
  r.rows = l.rows;
  r.ldc = l.ldc;
  r.rows_pad = l.rows_pad;
  r.tiles = (int)((c.V + l.width - 1) / l.width);
  r.part32 = l.part32;
  r.ld32 = l.ld32;
  r.k_piece = (int)(l.cut.piece / BK);
  r.part_room = l.cut.part_room;
  r.tile_rows = 128 * cg;
  r.twice = c.N <= TWICE;
  r.units = sms / cg;
  return r;
}

GemmArgs gemm_args(const Layout& l, bool twice, bool whole = false) {
  GemmArgs g = {};
  g.plan = l.plan;
  g.a_box = 128;
  g.twice = twice;
  g.whole = whole;
  g.target = l.packed;
  g.rows_pad = l.rows_pad;
  g.coef = l.coef;
  g.zt = l.zt;
  return g;
}

// Few rows: only the 32-row boxes that hold some are copied.
int a_box(int64_t N) { return N > 96 ? 128 : 32; }

// Packed rows and plan are there.  Statistics of all tiles, then the rows' losses.
template <int CG, bool BF16>
int forward(const Call& c, const Layout& l, RowArgs r, bool grads, Device dev, cudaStream_t st) {
  CUtensorMap rows, head;
  int rc = pesti_tensor_map(&rows, pesti_map_type(c.dtype), l.rows, c.D, l.rows_pad, l.ldc * 2, 64, a_box(c.N));
  if (!rc) rc = pesti_tensor_map(&head, pesti_map_type(c.dtype), c.head, c.D, c.V, c.w_ld * 2, 64, l.width / CG);
  if (rc) return rc;
  GemmArgs g = gemm_args(l, r.twice);
  g.width = l.width;
  g.m_tiles = -1;
  g.a_box = a_box(c.N);
  g.n_tiles = r.tiles;
  g.k_iters = (int)((c.D + BK - 1) / BK);
  g.fast_m = 1;
  g.V = (int)c.V;
  g.parts = l.parts;
  g.zsum = c.eps != 0.0 ? l.zsum : nullptr;
  rc = launch_gemm<CG, BF16, false, false, STATS>(rows, head, rows, g, dev, st);
  if (rc) return rc;
  r.parts = l.parts;
  r.zsum = g.zsum;
  const char* what = "lce_join_kernel launch";
  if (c.N <= 512)
    return launch(what, grads ? lce_join_kernel<1, true> : lce_join_kernel<1, false>, 1, dim3((unsigned)c.N), 256, 0,
                  st, r);
  return launch(what, grads ? lce_join_kernel<8, true> : lce_join_kernel<8, false>, 1, dim3((unsigned)((c.N + 7) / 8)),
                256, 0, st, r);
}

// Packed rows, plan and coefficients are there.
template <int CG, bool BF16>
int backward(const Call& c, const Layout& l, RowArgs r, void* dh, int64_t dh_ld, void* dw, int64_t dw_ld,
             Device dev, cudaStream_t st) {
  CUtensorMap rows_k, rows_mn, head_k, head_mn, out_w, out_h;
  int rc = pesti_tensor_map(&rows_k, pesti_map_type(c.dtype), l.rows, c.D, l.rows_pad, l.ldc * 2, 64, a_box(c.N));
  if (!rc) rc = pesti_tensor_map(&rows_mn, pesti_map_type(c.dtype), l.rows, c.D, l.rows_pad, l.ldc * 2, 64, 64);
  if (!rc) rc = pesti_tensor_map(&head_k, pesti_map_type(c.dtype), c.head, c.D, c.V, c.w_ld * 2, 64, BN / CG);
  if (!rc) rc = pesti_tensor_map(&head_mn, pesti_map_type(c.dtype), c.head, c.D, c.V, c.w_ld * 2, 64, 64);
  if (!rc && dw) rc = pesti_tensor_map(&out_w, pesti_map_type(c.dtype), dw, c.D, c.V, dw_ld * 2, 64, 32);
  if (!rc && dh) rc = pesti_tensor_map(&out_h, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, l.part32, c.D, l.cut.part_room, l.ld32 * 4, 32, 32);
  if (rc) return rc;
  const int d_tiles = (int)((c.D + BN - 1) / BN);
  for (long long v0 = 0; v0 < c.V; v0 += l.cut.piece) {
    const long long width = std::min<long long>(l.cut.piece, c.V - v0);
    CUtensorMap grad_out, grad_k, grad_mn;
    rc = pesti_tensor_map(&grad_out, pesti_map_type(c.dtype), l.grad, width, l.rows_pad, l.cut.piece * 2, 64, 32);
    if (!rc) rc = pesti_tensor_map(&grad_k, pesti_map_type(c.dtype), l.grad, width, l.rows_pad, l.cut.piece * 2, 64, a_box(c.N));
    if (!rc) rc = pesti_tensor_map(&grad_mn, pesti_map_type(c.dtype), l.grad, width, l.rows_pad, l.cut.piece * 2, 64, 64);
    if (rc) return rc;
    GemmArgs g = gemm_args(l, r.twice, !r.lse_in || r.nll_in);  // G of this piece
    g.m_tiles = -1;
    g.a_box = a_box(c.N);
    g.n_tiles = (int)((width + BN - 1) / BN);
    g.k_iters = (int)((c.D + BK - 1) / BK);
    g.fast_m = 1;
    g.v0 = (int)v0;
    g.b_row0 = (int)v0;
    g.V = (int)c.V;
    g.out_x = (int)width;
    g.out_y = (int)l.rows_pad;
    rc = launch_gemm<CG, BF16, false, false, GRAD>(rows_k, head_k, grad_out, g, dev, st);
    if (rc) return rc;
    if (dh) {  // dh += G W, first: this piece of the head is in L2 yet
      g = gemm_args(l, r.twice);
      g.m_tiles = -1;
      g.a_box = a_box(c.N);
      g.n_tiles = d_tiles;
      g.k_iters = (int)((width + BK - 1) / BK);
      g.b_k0 = v0;
      g.add = v0 != 0;
      g.out_x = (int)c.D;
      g.out_y = INT_MAX;
      rc = launch_gemm<CG, BF16, false, true, PART32>(grad_k, head_mn, out_h, g, dev, st);
      if (rc) return rc;
    }
    if (dw) {  // dW = G^T h
      g = gemm_args(l, r.twice);
      g.m_tiles = (int)((width + 128 * CG - 1) / (128 * CG));
      g.n_tiles = d_tiles;
      g.k_iters = -1;
      g.v0 = (int)v0;
      g.out_x = (int)c.D;
      g.out_y = (int)c.V;
      rc = launch_gemm<CG, BF16, true, true, OUT16>(grad_mn, rows_mn, out_w, g, dev, st);
      if (rc) return rc;
    }
  }
  if (!dh) return PESTI_OK;
  r.d_hidden = dh;
  r.dh_ld = dh_ld;
  const char* what = "lce_finish_kernel launch";
  if (c.N <= 256)
    return launch(what, lce_finish_kernel<BF16, 8>, 1, dim3((unsigned)((c.D + 127) / 128), (unsigned)c.N), 256, 0, st, r);
  // (rows beyond a grid's second dimension in further launches)
  for (long long n = 0; n < c.N; n += 65535) {
    RowArgs some = r;
    some.place += n;
    some.d_hidden = (char*)dh + n * dh_ld * 2;
    const dim3 grid((unsigned)((c.D + 1023) / 1024), (unsigned)std::min<long long>(65535, c.N - n));
    rc = launch(what, lce_finish_kernel<BF16, 1>, 1, grid, 256, 0, st, some);
    if (rc) return rc;
  }
  return PESTI_OK;
}

int backward(const Call& c, const Layout& l, const RowArgs& r, int cg, void* dh, int64_t dh_ld, void* dw, int64_t dw_ld,
             Device dev, cudaStream_t st) {
  const bool bf16 = c.dtype == PESTI_BF16;
  if (cg == 1) return (bf16 ? backward<1, true> : backward<1, false>)(c, l, r, dh, dh_ld, dw, dw_ld, dev, st);
  return (bf16 ? backward<2, true> : backward<2, false>)(c, l, r, dh, dh_ld, dw, dw_ld, dev, st);
}

template <bool BACKWARD>
int pack(const RowArgs& r, cudaStream_t st) {
  const char* what = "lce_pack_kernel launch";
  const dim3 rows((unsigned)r.rows_pad);
  if (r.N <= PACK_ROWS)
    return launch(what, lce_pack_kernel<BACKWARD, true>, 1, rows, (int)std::max<long long>(256, up_to(r.N, 32)), 0, st, r);
  const int rc = launch(what, lce_pack_kernel<BACKWARD, false>, 1, dim3(1), PACK_ROWS, 0, st, r);
  return rc ? rc : launch("lce_gather_kernel launch", lce_gather_kernel, 1, rows, 256, 0, st, r);
}

int check_scratch(const void* ws, int64_t have, long long need) {
  if (!ws || have < need) return refuse("workspace too small");
  if ((uintptr_t)ws % 256) return refuse("workspace is not 256-byte aligned");
  return PESTI_OK;
}

}  // namespace

extern "C" {

int64_t pesti_linear_ce_workspace(pesti_dtype dtype, int64_t N, int64_t V, int64_t D, int passes) {
  const int rc = check_sizes(dtype, N, V, D);
  if (rc) return rc;
  if (passes < 1 || passes > 3) return refuse("passes must be 1 to 3");
  return layout(nullptr, N, V, D, passes & 1, passes & 2).bytes;
}

int pesti_linear_ce(const void* d_hidden, pesti_dtype dtype, int64_t N, int64_t D, int64_t h_ld, const void* d_head,
                    int64_t V, int64_t w_ld, const void* d_target, int target_bytes, const float* d_weight,
                    double label_smoothing, double z_loss, float* d_loss, float* d_lse, void* d_grad_hidden,
                    int64_t gh_ld, void* d_grad_head, int64_t gw_ld, void* d_ws, int64_t ws_bytes, void* stream) {
  return pesti_linear_ce_nll(d_hidden, dtype, N, D, h_ld, d_head, V, w_ld, d_target, target_bytes, d_weight,
                             label_smoothing, z_loss, d_loss, d_lse, nullptr, d_grad_hidden, gh_ld, d_grad_head, gw_ld,
                             d_ws, ws_bytes, stream);
}

int pesti_linear_ce_backward(const void* d_hidden, pesti_dtype dtype, int64_t N, int64_t D, int64_t h_ld,
                             const void* d_head, int64_t V, int64_t w_ld, const void* d_target, int target_bytes,
                             const float* d_weight, double label_smoothing, double z_loss, const float* d_lse,
                             const float* d_up, int64_t up_stride, void* d_grad_hidden, int64_t gh_ld,
                             void* d_grad_head, int64_t gw_ld, void* d_ws, int64_t ws_bytes, void* stream) {
  return pesti_linear_ce_nll_backward(d_hidden, dtype, N, D, h_ld, d_head, V, w_ld, d_target, target_bytes, d_weight,
                                      label_smoothing, z_loss, d_lse, nullptr, d_up, up_stride, d_grad_hidden, gh_ld,
                                      d_grad_head, gw_ld, d_ws, ws_bytes, stream);
}

int pesti_linear_ce_nll(const void* d_hidden, pesti_dtype dtype, int64_t N, int64_t D, int64_t h_ld,
                        const void* d_head, int64_t V, int64_t w_ld, const void* d_target, int target_bytes,
                        const float* d_weight, double label_smoothing, double z_loss, float* d_loss, float* d_lse,
                        float* d_nll, void* d_grad_hidden, int64_t gh_ld, void* d_grad_head, int64_t gw_ld, void* d_ws,
                        int64_t ws_bytes, void* stream) {
  const Call c = {d_hidden, dtype, N, D, h_ld, d_head, V, w_ld, d_target, target_bytes, d_weight, label_smoothing,
                  z_loss};
  int rc = check(c);
  if (rc) return rc;
  if (N == 0 && !d_grad_head) return PESTI_OK;
  if (N && !d_loss) return refuse("null loss");
  if ((uintptr_t)d_loss % 4 || (uintptr_t)d_lse % 4 || (uintptr_t)d_nll % 4)
    return refuse("loss or lse is not aligned to its type");
  const bool grads = d_grad_hidden || d_grad_head;
  if (grads) {
    rc = check_grads(c, d_grad_hidden, gh_ld, d_grad_head, gw_ld);
    if (rc) return rc;
  }
  Device dev = {};
  cudaStream_t st = (cudaStream_t)stream;
  if (N == 0) {
    rc = pesti_current_device(dev.index, dev.sms);
    if (rc) return rc;
    const cudaError_t e = cudaMemset2DAsync(d_grad_head, gw_ld * 2, 0, D * 2, V, st);
    return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, "cudaMemset2DAsync");
  }
  rc = check_scratch(d_ws, ws_bytes, layout(nullptr, N, V, D, true, grads).bytes);
  if (rc) return rc;
  rc = pesti_current_device(dev.index, dev.sms);
  if (rc) return rc;
  const Layout l = layout((char*)d_ws, N, V, D, true, grads);
  const int cg = blocks_per_tile(N);
  RowArgs r = row_args(c, l, cg, dev.sms);
  r.loss = d_loss;
  r.lse = d_lse;
  r.nll = d_nll;
  rc = pack<false>(r, st);
  if (rc) return rc;
  const bool bf16 = dtype == PESTI_BF16;
  rc = cg == 1 ? (bf16 ? forward<1, true> : forward<1, false>)(c, l, r, grads, dev, st)
               : (bf16 ? forward<2, true> : forward<2, false>)(c, l, r, grads, dev, st);
  if (rc || !grads) return rc;
  return backward(c, l, r, cg, d_grad_hidden, gh_ld, d_grad_head, gw_ld, dev, st);
}

int pesti_linear_ce_nll_backward(const void* d_hidden, pesti_dtype dtype, int64_t N, int64_t D, int64_t h_ld,
                                 const void* d_head, int64_t V, int64_t w_ld, const void* d_target, int target_bytes,
                                 const float* d_weight, double label_smoothing, double z_loss, const float* d_lse,
                                 const float* d_nll, const float* d_up, int64_t up_stride, void* d_grad_hidden,
                                 int64_t gh_ld, void* d_grad_head, int64_t gw_ld, void* d_ws, int64_t ws_bytes,
                                 void* stream) {
  const Call c = {d_hidden, dtype, N, D, h_ld, d_head, V, w_ld, d_target, target_bytes, d_weight, label_smoothing,
                  z_loss};
  int rc = check(c);
  if (rc) return rc;
  if (up_stride < 0) return refuse("negative stride");
  if (!d_grad_hidden && !d_grad_head) return refuse("no gradient is asked for");
  if (N == 0 && !d_grad_head) return PESTI_OK;
  if (N && (!d_lse || !d_up)) return refuse("null lse or upstream gradient");
  if ((uintptr_t)d_lse % 4 || (uintptr_t)d_nll % 4 || (uintptr_t)d_up % 4)
    return refuse("lse or upstream gradient is not aligned to its type");
  rc = check_grads(c, d_grad_hidden, gh_ld, d_grad_head, gw_ld);
  if (rc) return rc;
  Device dev = {};
  cudaStream_t st = (cudaStream_t)stream;
  if (N == 0) {
    rc = pesti_current_device(dev.index, dev.sms);
    if (rc) return rc;
    const cudaError_t e = cudaMemset2DAsync(d_grad_head, gw_ld * 2, 0, D * 2, V, st);
    return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, "cudaMemset2DAsync");
  }
  rc = check_scratch(d_ws, ws_bytes, layout(nullptr, N, V, D, false, true).bytes);
  if (rc) return rc;
  rc = pesti_current_device(dev.index, dev.sms);
  if (rc) return rc;
  const Layout l = layout((char*)d_ws, N, V, D, false, true);
  const int cg = blocks_per_tile(N);
  RowArgs r = row_args(c, l, cg, dev.sms);
  r.lse_in = d_lse;
  r.nll_in = d_nll;
  r.up = d_up;
  r.up_stride = up_stride;
  rc = pack<true>(r, st);
  if (rc) return rc;
  return backward(c, l, r, cg, d_grad_hidden, gh_ld, d_grad_head, gw_ld, dev, st);
}

int pesti_testing_give_up(int product, int round) {
  if (product < 0 || product > PESTI_Q4_SUMS || round < -1) return refuse("product must be 0 to 4, round -1 or more");
  pesti_give_up_at.store((int64_t)product << 32 | (uint32_t)round, std::memory_order_relaxed);
  return PESTI_OK;
}

}  // extern "C"
