// Host side of the beam search entry points (include/pesti_sampler.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <vector>

#include "../../include/pesti_sampler.h"
#include "../../include/pesti_testing.h"
#include "pesti_beam.cuh"
#include "pesti_error.h"

namespace {

using namespace pesti_rows;

int refuse(const char* msg) { return pesti_set_error(PESTI_E_INVALID_ARG, msg); }

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

long long units_of(pesti_dtype dtype, long long V) {
  return dtype == PESTI_F32 ? row_units<float>(V) : row_units<__half>(V);
}

int check_sizes(pesti_dtype dtype, int64_t G, int64_t W, int64_t V, int64_t K) {
  if (dtype != PESTI_F32 && dtype != PESTI_BF16 && dtype != PESTI_F16)
    return refuse("logits must be f32, bf16 or f16");
  if (G < 0) return refuse("G < 0");
  if (W < 1 || W > PESTI_BEAM_MAX_WIDTH) return refuse("W must be 1 to 64");
  if (K < 1 || K > PESTI_BEAM_MAX_CAND) return refuse("K must be 1 to 128");
  if (V < 1 || V > 0x7fffffffLL) return refuse("V must be 1 to 2^31-1");
  // a block of the scan takes SCAN_WARPS units; the pick has at most a block per beam
  const long long per_row = (units_of(dtype, V) + SCAN_WARPS - 1) / SCAN_WARPS;
  if (G > 0x7fffffffLL / W / per_row) return refuse("G * W * V too large");
  return PESTI_OK;
}

long long up256(long long n) { return (n + 255) / 256 * 256; }

// Lays the scratch out behind `base` (which may be null, for the size alone).
long long layout(char* base, long long rows, long long units, BeamWs* ws) {
  const long long unit = up256(rows * units * (long long)sizeof(float2));
  if (ws) {
    ws->unit = (float2*)base;
    ws->seg = (uint32_t*)(base + unit);
  }
  return unit + up256(rows * units * UNIT_VECS * (long long)sizeof(uint32_t));
}

constexpr int kMaxDevices = 64;
constexpr int kPickSmem = 200 * 1024;  // most of a block's dynamic shared memory
std::atomic<int> g_pick_sms[kMaxDevices];  // 0: not set up yet

template <typename T, int TW>
cudaError_t allow_teams() {
  const cudaError_t e =
      cudaFuncSetAttribute(beam_pick_kernel<T, TW, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPickSmem);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(beam_pick_kernel<T, TW, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPickSmem);
}

template <typename T>
cudaError_t allow_pick() {
  cudaError_t e = allow_teams<T, 7>();
  if (e == cudaSuccess) e = allow_teams<T, 3>();
  return e == cudaSuccess ? allow_teams<T, 1>() : e;
}

int set_up_pick(int* sms) {
  int dev = 0, have = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return pesti_set_cuda_error(e, "cudaGetDevice");
  if (dev >= kMaxDevices) return refuse("device index out of range");
  *sms = g_pick_sms[dev].load(std::memory_order_acquire);
  if (*sms) return PESTI_OK;
  e = cudaDeviceGetAttribute(&have, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = allow_pick<float>();
  if (e == cudaSuccess) e = allow_pick<__nv_bfloat16>();
  if (e == cudaSuccess) e = allow_pick<__half>();
  if (e != cudaSuccess) return pesti_set_cuda_error(e, "beam_pick_kernel set-up");
  g_pick_sms[dev].store(have, std::memory_order_release);
  *sms = have;
  return PESTI_OK;
}

// Beams at a time in a block of teams of TW warps, and the blocks of a group.
void pick_shape(PickPlan& pl, int tw, long long* c) {
  const int most = PICK_WARPS / (tw + 1);
  *c = std::min<long long>(MAX_PICK_CLUSTER, (pl.W + most - 1) / most);
  pl.rows = (int)((pl.W + *c - 1) / *c);
  *c = (pl.W + pl.rows - 1) / pl.rows;
  pl.teams = std::min(pl.rows, most);
}

// Blocks of a group, and a block's dynamic shared memory.
struct PickLaunch {
  long long blocks, bytes;
};

// The plan for teams of `tw` warps; W, K and units are set.
PickLaunch plan_pick(PickPlan& pl, int tw) {
  PickLaunch to;
  pick_shape(pl, tw, &to.blocks);
  // A list takes what one round of a team's segments appends to a pruned one.
  // Longer rows have keys of runs of segments (empty ones at the end, so that
  // their number is a multiple of 4: the histogram behind them is read 16 bytes
  // at a time).
  const long long nseg = pl.units * UNIT_VECS, lists = list_bytes(pl.W, pl.K);
  pl.cap = RANK_CAP + tw * 256;
  const long long most = ((kPickSmem - lists) / pl.teams / 4 - (2 * pl.cap + TEAM_WORDS + 4)) / 4 * 4;
  pl.run = (int)((nseg + most - 1) / most);
  pl.nkeys = (int)(((nseg + pl.run - 1) / pl.run + 3) / 4 * 4);
  to.bytes = lists + std::max(pl.teams * team_bytes(pl.nkeys, pl.cap), lists);
  return to;
}

template <typename T, int TW>
int launch_pick(const void* logits, long long G, long long V, long long ld, PickPlan pl, const float* cum,
                const uint8_t* done, const BeamWs& ws, float* score, int32_t* token, int32_t* parent, float* lse,
                cudaStream_t st) {
  const PickLaunch to = plan_pick(pl, TW);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(G * to.blocks));
  cfg.blockDim = dim3((unsigned)(pl.teams * (TW + 1) * 32));
  cfg.dynamicSmemBytes = (size_t)to.bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)to.blocks;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(
      &cfg, pl.run == 1 ? beam_pick_kernel<T, TW, false> : beam_pick_kernel<T, TW, true>, (const T*)logits, ld, V,
      (const PickPlan)pl, cum, done, ws, score, token, parent, lse);
  return e == cudaSuccess ? PESTI_OK : pesti_set_cuda_error(e, "beam_pick_kernel launch");
}

// The widest teams whose blocks all run at once (16 warps of 114 registers
// fill an SM): 32 groups of 8 beams take 11.5 us with teams of 7, 16 us with
// teams of 3; 64 groups 21.5 us with teams of 7, 13 us with teams of 3.  Long
// lists are too much for teams of one warp (1024 rows of 32000, K 64: 73 us,
// 47 us with teams of 3); shorter ones are not (whole calls with teams of one
// and of 3: 128 groups of 8 x 32000 bf16, K 16 35 and 39 us; 256 groups of 8 x
// 32000 f32 82 and 92 us; 64 groups of 16 x 32000 bf16, K 32 51 and 55 us; only
// single beams of K 32 59 and 53 us).  Where teams of 7 fit, the blocks are not wanted
// for other groups and stay for rows to add up again: that costs every call
// 0.2 us, and brings two rows of 152064 f32 from 185 to 39 us.
int team_warps(PickPlan& pl, long long G, int sms) {
  auto at_once = [&](int tw) {
    long long c;
    PickPlan q = pl;
    pick_shape(q, tw, &c);
    return G * c * q.teams * (tw + 1) <= (long long)sms * PICK_WARPS;
  };
  pl.stay = at_once(7);
  return pl.stay ? 7 : at_once(3) || pl.K > 32 ? 3 : 1;
}

template <typename T>
int run_select(const void* logits, long long G, long long W, long long V, long long ld, const float* cum,
               const uint8_t* done, int K, float* score, int32_t* token, int32_t* parent, float* lse,
               const BeamWs& ws, long long units, cudaStream_t st) {
  int sms = 0;
  int rc = set_up_pick(&sms);
  if (rc) return rc;
  const long long per_row = (units + SCAN_WARPS - 1) / SCAN_WARPS;
  beam_scan_kernel<T><<<(unsigned)(G * W * per_row), SCAN_WARPS * 32, 0, st>>>(
      (const T*)logits, ld, V, (int)W, units, per_row, cum, done, lse != nullptr, ws);
  rc = launched("beam_scan_kernel launch");
  if (rc) return rc;
  PickPlan pl{};
  pl.W = (int)W;
  pl.K = K;
  pl.units = units;
  switch (team_warps(pl, G, sms)) {
    case 7: return launch_pick<T, 7>(logits, G, V, ld, pl, cum, done, ws, score, token, parent, lse, st);
    case 3: return launch_pick<T, 3>(logits, G, V, ld, pl, cum, done, ws, score, token, parent, lse, st);
    default: return launch_pick<T, 1>(logits, G, V, ld, pl, cum, done, ws, score, token, parent, lse, st);
  }
}

int check_state(const pesti_beam_state* s, int64_t G, int64_t W) {
  if (!s) return refuse("null beam state");
  if (G < 0 || G > 0x7fffffffLL) return refuse("G must be 0 to 2^31-1");
  if (W < 1 || W > PESTI_BEAM_MAX_WIDTH) return refuse("W must be 1 to 64");
  if (s->cap < 0 || s->cap > 0x7fffffffLL) return refuse("cap must be 0 to 2^31-1");
  if (G > 0 && (!s->cum || !s->last || !s->parent || !s->count || !s->done || !s->fin_len || !s->fin_score ||
                !s->fin_count || (s->cap > 0 && (!s->tokens || !s->fin_tokens))))
    return refuse("null array in the beam state");
  return PESTI_OK;
}

BeamStatePtrs pointers(const pesti_beam_state& s) {
  return BeamStatePtrs{s.cum,        s.last,    s.parent,    s.tokens,    s.count, s.done,
                       s.fin_tokens, s.fin_len, s.fin_score, s.fin_count, s.cap};
}

// Bytes from a state's first byte to behind its last one; -1 if they overflow.
long long extent(long long rows, long long row_stride, long long blocks, long long blk_stride, long long bytes) {
  const __int128 n = (__int128)(rows - 1) * row_stride + (__int128)(blocks - 1) * blk_stride + bytes;
  return n > (__int128)LLONG_MAX ? -1 : (long long)n;
}

template <typename Vec, int WB>
int launch_reorder(const ReorderArgs& a, long long tiles, const int32_t* parent, int W, cudaStream_t st) {
  beam_reorder_kernel<Vec, WB><<<(unsigned)tiles, REORDER_THREADS, 0, st>>>(a, parent, W);
  return launched("beam_reorder_kernel launch");
}

// Vector widths: 16 bytes for up to 16 beams (a thread holds every beam's
// vector in registers), 4 bytes beyond that, 1 byte where nothing is aligned.
int vec_bytes(const pesti_beam_rows& s, int W) {
  const unsigned long long bits = (unsigned long long)(uintptr_t)s.src | (unsigned long long)(uintptr_t)s.dst |
                                  (unsigned long long)s.src_row_stride | (unsigned long long)s.dst_row_stride |
                                  (unsigned long long)(s.blocks > 1 ? s.src_block_stride | s.dst_block_stride : 0) |
                                  (unsigned long long)s.block_bytes;
  if (W <= 16 && bits % 16 == 0) return 16;
  return bits % 4 == 0 ? 4 : 1;
}

// Tiles of a group.
__int128 reorder_tiles(const pesti_beam_rows& s, int vec) {
  return (__int128)((s.block_bytes / vec + REORDER_THREADS - 1) / REORDER_THREADS) * s.blocks;
}

int flush_reorder(ReorderArgs& a, long long& tiles, int vec, const int32_t* parent, int W, cudaStream_t st) {
  if (a.n == 0) return PESTI_OK;
  int rc;
  if (vec == 16)
    rc = W <= 4   ? launch_reorder<uint4, 4>(a, tiles, parent, W, st)
         : W <= 8 ? launch_reorder<uint4, 8>(a, tiles, parent, W, st)
                  : launch_reorder<uint4, 16>(a, tiles, parent, W, st);
  else if (vec == 4)
    rc = W <= 16 ? launch_reorder<uint32_t, 16>(a, tiles, parent, W, st)
                 : launch_reorder<uint32_t, 64>(a, tiles, parent, W, st);
  else
    rc = launch_reorder<uint8_t, 64>(a, tiles, parent, W, st);
  a.n = 0;
  tiles = 0;
  return rc;
}

}  // namespace

extern "C" {

int64_t pesti_beam_select_workspace(pesti_dtype dtype, int64_t G, int64_t W, int64_t V, int64_t K) {
  const int rc = check_sizes(dtype, G, W, V, K);
  if (rc) return rc;
  return layout(nullptr, G * W, units_of(dtype, V), nullptr);
}

int pesti_beam_select(const void* d_logits, pesti_dtype dtype, int64_t G, int64_t W, int64_t V, int64_t ld,
                      const float* d_cum, const uint8_t* d_done, int64_t K, float* d_score, int32_t* d_token,
                      int32_t* d_parent, float* d_lse, void* d_ws, int64_t ws_bytes, void* stream) {
  int rc = check_sizes(dtype, G, W, V, K);
  if (rc) return rc;
  if (ld < V) return refuse("ld is below V");
  if (G == 0) return PESTI_OK;
  if (!d_logits) return refuse("null logits");
  if (!d_score || !d_token || !d_parent) return refuse("null output");
  if ((uintptr_t)d_logits % (dtype == PESTI_F32 ? 4 : 2)) return refuse("logits are not aligned to their type");
  const long long units = units_of(dtype, V);
  BeamWs ws;
  const long long need = layout((char*)d_ws, G * W, units, &ws);
  if (!d_ws || ws_bytes < need) return refuse("workspace too small");
  if ((uintptr_t)d_ws % 256) return refuse("workspace is not 256-byte aligned");
  rc = need_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == PESTI_BF16)
    return run_select<__nv_bfloat16>(d_logits, G, W, V, ld, d_cum, d_done, (int)K, d_score, d_token, d_parent, d_lse,
                                     ws, units, st);
  if (dtype == PESTI_F16)
    return run_select<__half>(d_logits, G, W, V, ld, d_cum, d_done, (int)K, d_score, d_token, d_parent, d_lse, ws,
                              units, st);
  return run_select<float>(d_logits, G, W, V, ld, d_cum, d_done, (int)K, d_score, d_token, d_parent, d_lse, ws, units,
                           st);
}

int pesti_testing_beam_plan(pesti_dtype dtype, int64_t G, int64_t W, int64_t V, int64_t K, int sms,
                            pesti_testing_plan* plan) {
  const int rc = check_sizes(dtype, G, W, V, K);
  if (rc) return rc;
  if (!plan) return refuse("null plan");
  PickPlan pl{};
  pl.W = (int)W;
  pl.K = (int)K;
  pl.units = units_of(dtype, V);
  const int tw = team_warps(pl, G, sms);
  const PickLaunch to = plan_pick(pl, tw);
  plan->segments = pl.units * UNIT_VECS;
  plan->team_warps = tw;
  plan->teams = pl.teams;
  plan->blocks = to.blocks;
  plan->stay = pl.stay;
  plan->run = pl.run;
  plan->keys = pl.nkeys;
  plan->team_at = list_bytes(pl.W, pl.K);
  plan->team_stride = team_bytes(pl.nkeys, pl.cap);
  plan->keys_at = keys_offset(pl.cap);
  plan->hist_at = hist_offset(pl.nkeys, pl.cap);
  plan->bytes = to.bytes;
  plan->most_bytes = kPickSmem;
  return PESTI_OK;
}

int pesti_beam_reset(const pesti_beam_state* state, int64_t G, int64_t W, void* stream) {
  int rc = check_state(state, G, W);
  if (rc) return rc;
  if (G == 0) return PESTI_OK;
  rc = need_device();
  if (rc) return rc;
  const long long n = std::max((long long)G * W * state->cap, (long long)G * W);
  const long long blocks = std::min(1184LL, (n + 255) / 256);
  beam_reset_kernel<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(G, (int)W, pointers(*state));
  return launched("beam_reset_kernel launch");
}

int pesti_beam_advance(const pesti_beam_state* state, const float* d_score, const int32_t* d_token,
                       const int32_t* d_parent, int64_t G, int64_t W, int64_t K, const uint32_t* d_stop,
                       int64_t n_stop, const pesti_beam_limits* limits, void* stream) {
  int rc = check_state(state, G, W);
  if (rc) return rc;
  if (!limits) return refuse("null limits");
  if (K < 1 || K > PESTI_BEAM_MAX_CAND) return refuse("K must be 1 to 128");
  if (n_stop < 0) return refuse("n_stop < 0");
  if (limits->max_tokens < 0 || limits->max_seq_len < 0) return refuse("max_tokens or max_seq_len < 0");
  if (limits->max_tokens > 0x7fffffffLL || limits->max_seq_len > 0x7fffffffLL)
    return refuse("limits exceed 2^31-1");
  if (!std::isfinite(limits->length_penalty)) return refuse("length_penalty is not finite");
  if (state->cap < std::min(limits->max_tokens, limits->max_seq_len))
    return refuse("cap is below min(max_tokens, max_seq_len)");
  if (G == 0) return PESTI_OK;
  if (!d_score || !d_token || !d_parent) return refuse("null candidates");
  if (n_stop > 0 && !d_stop) return refuse("null stop list");
  rc = need_device();
  if (rc) return rc;
  const size_t smem = (size_t)W * ADV_THREADS * sizeof(int32_t);
  beam_advance_kernel<<<(unsigned)G, ADV_THREADS, smem, (cudaStream_t)stream>>>(
      d_score, d_token, d_parent, (int)W, (int)K, d_stop, n_stop, limits->max_tokens, limits->max_seq_len,
      limits->length_penalty, limits->early_stop != 0, pointers(*state));
  return launched("beam_advance_kernel launch");
}

int pesti_beam_reorder(const pesti_beam_rows* states, int64_t n_states, const int32_t* d_parent, int64_t G,
                       int64_t W, void* stream) {
  if (n_states < 0 || G < 0) return refuse("n_states or G < 0");
  if (W < 1 || W > PESTI_BEAM_MAX_WIDTH) return refuse("W must be 1 to 64");
  if (n_states > 0 && !states) return refuse("null states");
  if (G > LLONG_MAX / W / (long long)sizeof(int32_t)) return refuse("G * W too large");
  for (int64_t i = 0; i < n_states; ++i) {
    const pesti_beam_rows& s = states[i];
    if (s.blocks < 0 || s.block_bytes < 0) return refuse("blocks or block_bytes < 0");
    if (s.src_row_stride < 0 || s.dst_row_stride < 0 || s.src_block_stride < 0 || s.dst_block_stride < 0)
      return refuse("negative stride");
    if (G == 0 || s.blocks == 0 || s.block_bytes == 0) continue;
    if (!s.src || !s.dst) return refuse("null state");
    const long long a = extent(G * W, s.src_row_stride, s.blocks, s.src_block_stride, s.block_bytes);
    const long long b = extent(G * W, s.dst_row_stride, s.blocks, s.dst_block_stride, s.block_bytes);
    if (a < 0 || b < 0) return refuse("state too large");
    // a row's blocks and the rows must not share bytes where they are written
    if (s.blocks > 1 && s.dst_block_stride < s.block_bytes) return refuse("blocks of a row overlap");
    const long long one = extent(1, 0, s.blocks, s.dst_block_stride, s.block_bytes);
    if (G * W > 1 && s.dst_row_stride < s.block_bytes) return refuse("rows overlap");
    if (G * W > 1 && s.blocks > 1 && s.dst_row_stride < one) {
      // blocks outside rows (e.g. [heads, rows, dim]): every row fits between two blocks
      if (extent(G * W, s.dst_row_stride, 1, 0, s.block_bytes) > s.dst_block_stride) return refuse("rows overlap");
    }
    const char *p = (const char*)s.src, *q = (const char*)s.dst;
    if (p == q) {
      if (s.src_row_stride != s.dst_row_stride || (s.blocks > 1 && s.src_block_stride != s.dst_block_stride))
        return refuse("in-place states need equal strides");
    } else if (p < q + b && q < p + a) {
      return refuse("src and dst overlap");
    }
    // refused before anything is launched
    if (reorder_tiles(s, vec_bytes(s, (int)W)) * G > 0x7fffffff) return refuse("state too large");
  }
  if (G == 0 || n_states == 0) return PESTI_OK;
  // a state given twice would be moved twice
  if (n_states > 1) {
    try {
      std::vector<const void*> dsts;
      for (int64_t i = 0; i < n_states; ++i)
        if (states[i].blocks > 0 && states[i].block_bytes > 0) dsts.push_back(states[i].dst);
      std::sort(dsts.begin(), dsts.end());
      if (std::adjacent_find(dsts.begin(), dsts.end()) != dsts.end()) return refuse("a state is given twice");
    } catch (...) {
      return refuse("too many states");
    }
  }
  if (!d_parent) return refuse("null parents");
  // every block reads the parents, some behind others' writes
  for (int64_t i = 0; i < n_states; ++i) {
    const pesti_beam_rows& s = states[i];
    if (s.blocks == 0 || s.block_bytes == 0) continue;
    const char *p = (const char*)d_parent, *q = (const char*)s.dst;
    const long long b = extent(G * W, s.dst_row_stride, s.blocks, s.dst_block_stride, s.block_bytes);
    if (p < q + b && q < p + G * W * (long long)sizeof(int32_t)) return refuse("the parents overlap a state");
  }
  int rc = need_device();
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  for (const int vec : {16, 4, 1}) {
    ReorderArgs a;
    a.n = 0;
    long long tiles = 0;
    for (int64_t i = 0; i < n_states; ++i) {
      const pesti_beam_rows& s = states[i];
      if (s.blocks == 0 || s.block_bytes == 0 || vec_bytes(s, (int)W) != vec) continue;
      const long long vecs = s.block_bytes / vec, per = (vecs + REORDER_THREADS - 1) / REORDER_THREADS;
      const long long mine = per * s.blocks * G;
      if (a.n == REORDER_MAX || tiles + mine > 0x7fffffffLL) {
        rc = flush_reorder(a, tiles, vec, d_parent, (int)W, st);
        if (rc) return rc;
      }
      a.s[a.n++] = ReorderState{(const char*)s.src, (char*)s.dst,       s.src_row_stride,
                                s.dst_row_stride,   s.src_block_stride, s.dst_block_stride,
                                vecs,               per,                s.blocks,
                                tiles};
      tiles += mine;
    }
    rc = flush_reorder(a, tiles, vec, d_parent, (int)W, st);
    if (rc) return rc;
  }
  return PESTI_OK;
}

}  // extern "C"
