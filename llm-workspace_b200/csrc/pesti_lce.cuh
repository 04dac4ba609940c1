// Cross entropy from hidden states, without keeping the logits (pesti_linear_ce*).
//
//   z = h W^T,  lse = log sum exp z,  loss = a [lse - (1 - eps) z_t - eps mean(z) + zeta lse^2]
//   G = dloss/dz = c1 p - c2 [v = t] - c3,  c1 = a up (1 + 2 zeta lse), c2 = a up (1 - eps), c3 = a up eps / V
//   dh = G W,  dW = G^T h
//
// Where p_t is near 1, neither lse - z_t nor c1 p_t - c2 is left much of in f32.  So a row's other logits are summed
// without the target's, and from r = (their sum) / exp z_t come
//   -log p_t = log(1 + r),  G_t = a up [(1 + 2 zeta lse) (p_t - 1) + 2 zeta lse + eps - eps / V],  p_t - 1 = -r / (1 + r)
// as exact, relative to themselves, as r is.
//
// Three products of one size each way, and the logits' product again, since they are not kept: 8 N V D operations
// with gradients.  All four run in head_gemm_kernel, which differs in its operands' majors and in what becomes of the
// accumulators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>

#include "pesti_common.cuh"
#include "pesti_umma.cuh"

namespace pesti_lce {

using namespace pesti_umma;

constexpr int BN = 256;              // columns of a tile
constexpr int BK = 64;               // of K per stage: one 128-byte swizzled row
constexpr int EPI_WARPS = 8;         // a quarter of the accumulators' 128 rows and half of their columns each
constexpr int HALF = BN / 2;
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr int A_BYTES = 128 * BK * 2;
constexpr int OUT_BYTES = 32 * 128;  // a warp's 32 rows of 128 bytes on their way out
// Stages that logits are summed over in the tensor cores at once; the sums of several are added in registers.  The
// cores' own sums are cut off and not rounded, every 16 of K, and always towards 0: over 4096 of K that shrank the
// largest logits by 5e-6 of themselves, four times as much as in parts of 1024.  The gradients' logits are summed in the
// same parts: p = exp(z - lse) takes its logits to be the very ones that lse was made from.  (Cut otherwise, they left a
// target's p too small by 1e-4 of itself, which is all of 1 - p of a row with p = 0.9999.)
constexpr int PART_K = 16;
constexpr float LOG2E = 1.44269504f;

__host__ __device__ constexpr int b_bytes(int cg) { return BN / cg * BK * 2; }

// What the host does not know: written by the plan kernel, on the device.
struct Plan {
  int active;     // rows with a target and a weight
  unsigned gmax;  // bits of an f32 that no |G| of a row with finite coefficients exceeds (f16 only)
  int splits;     // ranges of K in the hidden states' gradient
  int part_rows;  // rows of a range's part: the active ones, to a whole tile
  int failed;     // a wait gave up: what is made behind it is NaN
};

struct RowCoef {
  float c, c1, c3;  // p = 2^(z log2e - c)
  float target;     // G_t, or what p_t's part of it lacks, -c2
};

enum Epilogue { STATS, GRAD, OUT16, PART32 };

// Up to this many rows G is held as a sum of two 16-bit values, the second in rows TWICE behind the first, and the packed
// rows are there twice.  A tile has 128 rows in any case, so that this costs a little writing, and few rows' gradients,
// which hang on few values of G, are as exact as their own type: a single row's were off by 2^-8 instead of 2^-9.
constexpr int TWICE = 64;

// Stages in shared memory, beside what is on its way out.
__host__ __device__ constexpr int out_bytes(Epilogue e) { return e == STATS ? 4096 : EPI_WARPS * 2 * OUT_BYTES; }
__host__ __device__ constexpr int stages(int cg, Epilogue e) {
  return (230000 - out_bytes(e)) / (A_BYTES + b_bytes(cg));
}
__host__ __device__ constexpr int smem_bytes(int cg, Epilogue e) {
  return 1024 + stages(cg, e) * (A_BYTES + b_bytes(cg)) + out_bytes(e) + 256;
}

struct GemmArgs {
  Plan* plan;
  int m_tiles, n_tiles;  // a negative count: from the active rows
  int k_iters;           // likewise
  int fast_m;            // the row tiles run fastest (else the column tiles)
  long long a_k0, b_k0;  // where K begins in A and B (rows of an MN-major operand, columns of a K-major one)
  int a_row0, b_row0;    // where the tiles' rows begin in A and B
  int a_box;             // rows of a copy of a K-major A: 128, or 32 where few rows count
  // STATS and GRAD
  const int* target;  // [rows], of the packed rows
  int v0, V;          // GRAD: the tiles' first token; the vocabulary
  float2* parts;      // [tiles, rows_pad] (maximum, sum) of a tile's logits but the target's, in powers of two
  float* zsum;        // [tiles, rows_pad] their plain sum, or null
  float* zt;          // [rows] the target's logit
  long long rows_pad;
  const RowCoef* coef;
  int whole;          // GRAD: the coefficients have G_t
  int add;            // PART32: add to what is there
  int out_x, out_y;   // where the output ends
  int width;          // columns of a tile (STATS: a multiple of 16)
  int twice;          // G and the packed rows are held twice
  int give_up;        // for tests: which of a block's tiles is taken for one whose wait gave up (-1: none)
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <bool BF16>
__device__ __forceinline__ float rounded(float x) {
  return BF16 ? __bfloat162float(__float2bfloat16_rn(x)) : __half2float(__float2half_rn(x));
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The power of two that brings |G| below 2^15: f16 holds p down to 2^-39 of the largest |G| then, and the scale is
// taken out of the sums exactly.  bf16 has the range of f32 and needs none.
template <bool BF16>
__device__ __forceinline__ int grad_shift(const Plan* plan) {
  if (BF16) return 0;
  const float m = __uint_as_float(plan->gmax);
  if (!(m > 0.0f)) return 0;
  return min(126, 14 - ilogbf(m));  // (-113 at least: the power and its inverse are both normal)
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// With 4096 rows x 128256 x 4096 each product runs at 521 clocks for a pair's 256 x 256 x 64, of the tensor cores' 512
// (1.37 PFLOP/s at the clock that the power limit leaves); with 16 rows the head passes at 6.1 TB/s.
// One block (CG 1) or a pair of them (CG 2) takes tiles of 128 CG x 256, one after another.  Warp 8 copies the stages
// in, one thread of warp 9 issues the products, warps 0 to 7 empty one set of accumulators while the other is filled.
template <int CG, bool BF16, bool A_MN, bool B_MN, Epilogue E>
__global__ void __launch_bounds__(THREADS, 1)
    head_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ CUtensorMap map_out, const GemmArgs g) {
  constexpr int ST = stages(CG, E), B_BYTES = b_bytes(CG), STAGE = A_BYTES + B_BYTES, TM = 128 * CG;
  extern __shared__ char raw[];
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t out0 = base + ST * STAGE;
  const uint32_t bars = out0 + out_bytes(E);
  const uint32_t full = bars, empty = bars + 8 * ST, acc_full = empty + 8 * ST, acc_empty = acc_full + 16,
                 given = acc_empty + 16, taken = given + 32;
  __shared__ uint32_t tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0 : cluster_rank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      bar_init(full + 8 * s, 1);
      bar_init(empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      bar_init(acc_full + 8 * s, 1);
      bar_init(acc_empty + 8 * s, CG * EPI_WARPS);
    }
    for (int s = 0; s < 8; ++s) bar_init(given + 8 * s, 1);  // given and taken, of each quarter
    bar_init_fence();
  }
  if (warp == EPI_WARPS + 1) tmem_alloc<CG>(smem_addr(&tmem_base), 512);
  fence_before();
  if constexpr (CG == 2) cluster_sync();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base;
  depend_wait();
  depend_launch();

  const int active = g.plan->active;
  const int m_tiles = g.m_tiles < 0 ? (active + TM - 1) / TM : g.m_tiles;
  const int n_tiles = g.n_tiles;
  const int k_rows = active && g.twice ? 2 * TWICE : active;
  const int k_iters = g.k_iters < 0 ? (k_rows + BK - 1) / BK : g.k_iters;
  const int splits = E == PART32 ? g.plan->splits : 1, k_split = (k_iters + splits - 1) / splits;
  const int per_split = m_tiles * n_tiles, tiles = per_split * splits;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  // tile -> (row tile, column tile, first stage of K, stages of K); 16 tiles of the fast side at a time
  auto locate = [&](int tile, int& m, int& n, int& split, int& k0, int& kn) {
    split = tile / per_split;
    const int r = tile - split * per_split;
    const int fast = g.fast_m ? m_tiles : n_tiles, slow = g.fast_m ? n_tiles : m_tiles;
    const int group = r / (16 * slow), at = r - group * 16 * slow, width = min(16, fast - group * 16);
    const int f = group * 16 + at % width, s = at / width;
    m = g.fast_m ? f : s;
    n = g.fast_m ? s : f;
    k0 = split * k_split;
    kn = max(0, min(k_split, k_iters - k0));
  };

  auto parts_of = [&](int kn) { return E == STATS || E == GRAD ? (kn + PART_K - 1) / PART_K : 1; };

  if (warp == EPI_WARPS) {
    if (elect_one()) {
      tma_prefetch(&map_a);
      tma_prefetch(&map_b);
      int s = 0, ph = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step) {
        int m, n, split, k0, kn;
        locate(tile, m, n, split, k0, kn);
        const int row_a = g.a_row0 + m * TM + (int)rank * 128;
        const int width = E == STATS ? g.width : BN;
        // rows of A that nothing comes of stay what they were in shared memory: they reach no row but their own
        const int rows_a = E == PART32 && g.twice ? 2 * TWICE : active;
        const int boxes = A_MN || g.a_box == 128 ? 1 : max(1, min(4, (rows_a - row_a + 31) / 32));
        const uint32_t bytes = CG * (A_MN || g.a_box == 128 ? A_BYTES : boxes * (A_BYTES / 4)) + width * BK * 2;
        const int row_b = g.b_row0 + n * width + (int)rank * (width / CG);
        for (int k = 0; k < kn; ++k) {
          if (!bar_wait(empty + 8 * s, ph ^ 1)) {
            ok = false;
            break;
          }
          const uint32_t bar = CG == 1 ? full + 8 * s : peer_addr(full + 8 * s, 0);
          if (rank == 0) bar_expect(full + 8 * s, bytes);
          const uint32_t a = base + s * STAGE, b = a + A_BYTES;
          const int ka = (int)(g.a_k0 + (long long)(k0 + k) * BK), kb = (int)(g.b_k0 + (long long)(k0 + k) * BK);
          if constexpr (A_MN) {
            for (int i = 0; i < 2; ++i) tma_load<CG>(a + i * 8192, &map_a, bar, row_a + 64 * i, ka);
          } else {
            for (int i = 0; i < boxes; ++i) tma_load<CG>(a + i * (A_BYTES / 4), &map_a, bar, ka, row_a + 32 * i);
          }
          if constexpr (B_MN) {
            for (int i = 0; i < 4 / CG; ++i) tma_load<CG>(b + i * 8192, &map_b, bar, row_b + 64 * i, kb);
          } else {
            tma_load<CG>(b, &map_b, bar, kb, row_b);  // a block's whole share of the tile
          }
          if (++s == ST) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // every stage is read, and the products' arrivals have reached this block
      for (int i = 0, at = s, at_ph = ph; i < ST && ok; ++i) {
        ok = bar_wait(empty + 8 * at, at_ph ^ 1);
        if (++at == ST) {
          at = 0;
          at_ph ^= 1;
        }
      }
      if (!ok) {
        atomicExch(&g.plan->failed, 1);
        for (int i = 0; i < ST && rank == 0; ++i) bar_wait(full + 8 * i, i < s ? ph : ph ^ 1);  // copies in flight
      }
    }
  } else if (warp == EPI_WARPS + 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t desc = mma_desc(BF16, A_MN, B_MN, TM, E == STATS ? g.width : BN);
      int s = 0, ph = 0, acc = 0, acc_ph = 0;
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step) {
        int m, n, split, k0, kn;
        locate(tile, m, n, split, k0, kn);
        const int parts = parts_of(kn);
        for (int part = 0; part < parts && ok; ++part) {
          if (!bar_wait(acc_empty + 8 * acc, acc_ph ^ 1)) {
            ok = false;
            break;
          }
          fence_after();
          const uint32_t d = tmem + acc * BN;
          const int k_end = kn * (part + 1) / parts, k_begin = kn * part / parts;
          for (int k = k_begin; k < k_end; ++k) {
            if (!bar_wait(full + 8 * s, ph)) {
              ok = false;
              break;
            }
            fence_after();
            const uint32_t a = base + s * STAGE, b = a + A_BYTES;
            const uint64_t da = operand_desc(a, 8192), db = operand_desc(b, 8192);
#pragma unroll
            for (int j = 0; j < BK / 16; ++j)  // 16 of K: 32 bytes of a row, or 16 rows of 128 bytes
              mma_f16<CG>(d, da + j * (A_MN ? 128 : 2), db + j * (B_MN ? 128 : 2), desc, k > k_begin || j > 0);
            mma_commit<CG>(empty + 8 * s);
            if (++s == ST) {
              s = 0;
              ph ^= 1;
            }
          }
          if (ok) mma_commit<CG>(acc_full + 8 * acc);
          acc ^= 1;
          if (acc == 0) acc_ph ^= 1;
        }
      }
      if (!ok) {
        atomicExch(&g.plan->failed, 1);
      }
    }
  } else {
    const int shift = (E == GRAD || E == OUT16) ? grad_shift<BF16>(g.plan) : 0;
    // (a wait that gave up in an earlier kernel makes NaN of what comes out)
    const float scale = g.plan->failed ? NAN : pow2(E == OUT16 ? -shift : shift);
    const int quarter = warp & 3, half0 = (warp >> 2) * HALF;
    const uint32_t out = out0 + warp * 2 * OUT_BYTES;  // two boxes
    const uint32_t row_out = out + lane * 128, swz = (lane & 7) << 4;
    const uint32_t acc_empty_to = CG == 1 ? acc_empty : peer_addr(acc_empty, 0);
    int acc = 0, acc_ph = 0, pair_ph = 0;
    // Once a wait has given up, kernels behind this one see it in the plan.  The head's gradient may be the last one: its
    // tiles from there on are written as NaN, without more waiting.  (`ok` is the same in all lanes.)
    bool ok = true;
    int round = 0;
    for (int tile = first; tile < tiles && (ok || E == OUT16); tile += step, ++round) {
      int m, n, split, k0, kn;
      locate(tile, m, n, split, k0, kn);
      const int warp_row = m * TM + (int)rank * 128 + quarter * 32, row = warp_row + lane;
      const int col0 = n * (E == STATS ? g.width : BN) + half0;
      auto wait_acc = [&]() {
        ok = __all_sync(PESTI_FULL_MASK, bar_wait(acc_full + 8 * acc, acc_ph)) && round != g.give_up;
        if (!ok) atomicExch(&g.plan->failed, 1);
        fence_after();
        return tmem + acc * BN + half0 + ((uint32_t)quarter << 21);
      };
      auto leave_acc = [&]() {
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_cluster(acc_empty_to + 8 * acc);
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1;
      };

      // the warp's accumulators, which are free for the next tile but one then
      float v[HALF];
      auto take_acc = [&]() {
        const uint32_t from = ok ? wait_acc() : 0;
        if (!ok) {
#pragma unroll
          for (int j = 0; j < HALF; ++j) v[j] = NAN;
          return;
        }
        uint32_t w[HALF];
#pragma unroll
        for (int c = 0; c < HALF; c += 32) tmem_load32(from + c, *(uint32_t(*)[32])(w + c));
        tmem_load_wait();
        leave_acc();
#pragma unroll
        for (int j = 0; j < HALF; ++j) v[j] = __uint_as_float(w[j]);
      };
      // the same of logits: the sums of their parts
      auto sum_acc = [&]() {
        const int parts = parts_of(kn);
#pragma unroll 1
        for (int part = 0; part < parts; ++part) {
          const uint32_t from = wait_acc();
          if (!ok) break;
#pragma unroll
          for (int c = 0; c < HALF; c += 32) {
            uint32_t w[32];
            tmem_load32(from + c, w);
            tmem_load_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[c + j] = __uint_as_float(w[j]) + (part ? v[c + j] : 0.0f);
          }
          leave_acc();
        }
      };
      // 128 bytes of each of the warp's rows in one of two boxes: written swizzled, so that eight lanes write to eight
      // banks' groups
      auto begin_out = [&]() {
        if (lane == 0) store_wait_read<0>();
        __syncwarp();
      };
      auto put16 = [&](int box, int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_out + box * OUT_BYTES +
                                                                      ((uint32_t)(chunk << 4) ^ swz)),
                     "r"(x), "r"(y), "r"(z), "r"(w)
                     : "memory");
      };
      auto end_out = [&](int x0, int x1, int y, bool add) {
        fence_smem_async();
        __syncwarp();
        if (lane == 0) {
#pragma unroll
          for (int box = 0; box < 2; ++box) {
            const int x = box ? x1 : x0;
            if (y >= g.out_y || x >= g.out_x) continue;
            if (add)
              tma_add(&map_out, out + box * OUT_BYTES, x, y);
            else
              tma_store(&map_out, out + box * OUT_BYTES, x, y);
          }
          store_commit();
        }
      };
      auto put_pairs = [&](int c) {  // 32 columns from c, in 16 bits
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack2<BF16>(v[c + 8 * j + 2 * i], v[c + 8 * j + 2 * i + 1]);
          put16(c / 64, c % 64 / 8 + j, w[0], w[1], w[2], w[3]);
        }
      };

      if constexpr (E == STATS) {
        const bool live = row < active;
        const int t = live ? g.target[row] - col0 : -1;
        sum_acc();
        float mx = -INFINITY, sum = 0.0f, zs = 0.0f, zt = 0.0f;
        const int left = min(g.V - col0, g.width - half0);  // columns of this half
#pragma unroll
        for (int c = 0; c < HALF; c += 32) {
          if (c >= left) continue;
          const bool here = __any_sync(PESTI_FULL_MASK, t >= c && t < c + 32);
          if (here) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (t == c + j) zt = v[c + j];
          }
          if (c + 32 > left) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j >= left) v[c + j] = -INFINITY;
          }
          if (g.zsum) {
            float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 32; ++j) a[j & 3] += c + j < left ? v[c + j] : 0.0f;
            zs += (a[0] + a[1]) + (a[2] + a[3]);
          }
          if (here) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (t == c + j) v[c + j] = -INFINITY;
          }
          float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 32; ++j) most[j & 3] = fmaxf(most[j & 3], v[c + j]);
          const float now = fmaxf(mx, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * LOG2E);
          const float ref = now == -INFINITY ? 0.0f : now;
          float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < 32; ++j) a[j & 3] += ex2(fmaf(v[c + j], LOG2E, -ref));
          sum = sum * ex2(mx - ref) + ((a[0] + a[1]) + (a[2] + a[3]));
          mx = now;
        }
        if (t >= 0 && t < min(HALF, left)) g.zt[row] = zt;
        // the tile's other half: its warp hands its sums over in shared memory
        float* other = (float*)(raw + (out0 - smem_addr(raw))) + quarter * 128 + lane;
        if (half0) {
          ok = ok && __all_sync(PESTI_FULL_MASK, bar_wait(taken + 8 * quarter, pair_ph ^ 1));
          other[0] = mx;
          other[32] = sum;
          other[64] = zs;
          __syncwarp();
          if (lane == 0) bar_arrive(given + 8 * quarter);
        } else {
          ok = ok && __all_sync(PESTI_FULL_MASK, bar_wait(given + 8 * quarter, pair_ph));
          const float m2 = other[0], s2 = other[32], z2 = other[64];
          __syncwarp();
          if (lane == 0) bar_arrive(taken + 8 * quarter);
          const float now = fmaxf(mx, m2), ref = now == -INFINITY ? 0.0f : now;
          if (live) {
            const long long at = (long long)n * g.rows_pad + row;
            g.parts[at] = make_float2(now, sum * ex2(mx - ref) + s2 * ex2(m2 - ref));
            if (g.zsum) g.zsum[at] = zs + z2;
          }
        }
        pair_ph ^= 1;
        if (!ok) atomicExch(&g.plan->failed, 1);
      } else if constexpr (E == GRAD) {
        sum_acc();
        const bool live = row < active;
        RowCoef k = {};
        int t = -1;
        if (live) {
          k = g.coef[row];
          t = g.target[row] - (g.v0 + col0);
        }
        const float c1 = k.c1 * scale, c3 = k.c3 * scale, target = k.target * scale;
        begin_out();
#pragma unroll
        for (int c = 0; c < HALF; c += 32) {
#pragma unroll
          for (int j = c; j < c + 32; ++j) {
            const float p = ex2(fmaf(v[j], LOG2E, -k.c));
            v[j] = fmaf(c1, p, -c3);
          }
          if (__any_sync(PESTI_FULL_MASK, t >= c && t < c + 32)) {
#pragma unroll
            for (int j = c; j < c + 32; ++j)
              if (t == j) v[j] = (g.whole ? 0.0f : v[j]) + target;
          }
          if (!live) {
#pragma unroll
            for (int j = c; j < c + 32; ++j) v[j] = 0.0f;
          }
          put_pairs(c);
        }
        if (!g.twice) {
          end_out(col0, col0 + 64, warp_row, false);
        } else if (warp_row < TWICE) {
          end_out(col0, col0 + 64, warp_row, false);
          begin_out();
#pragma unroll
          for (int c = 0; c < HALF; c += 32) {
#pragma unroll
            for (int j = c; j < c + 32; ++j) v[j] -= rounded<BF16>(v[j]);
            put_pairs(c);
          }
          end_out(col0, col0 + 64, TWICE + warp_row, false);
        }
      } else if constexpr (E == OUT16) {
        take_acc();
        begin_out();
#pragma unroll
        for (int c = 0; c < HALF; c += 32) {
#pragma unroll
          for (int j = c; j < c + 32; ++j) v[j] = kn ? v[j] * scale : 0.0f;
          put_pairs(c);
        }
        end_out(col0, col0 + 64, g.v0 + warp_row, false);
      } else {
        take_acc();
        if ((g.twice ? warp_row % TWICE : warp_row) < active) {
#pragma unroll
          for (int c = 0; c < HALF; c += 64) {
            begin_out();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int i = c + 4 * j;
              put16(j / 8, j % 8, kn ? __float_as_uint(v[i]) : 0u, kn ? __float_as_uint(v[i + 1]) : 0u,
                    kn ? __float_as_uint(v[i + 2]) : 0u, kn ? __float_as_uint(v[i + 3]) : 0u);
            }
            end_out(col0 + c, col0 + c + 32, split * g.plan->part_rows + warp_row, g.add != 0);
          }
        }
      }
    }
    if (lane == 0) store_wait_all();
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  fence_after();
  if (warp == EPI_WARPS + 1) tmem_free<CG>(tmem, 512);
}

struct RowArgs {
  Plan* plan;
  const void* hidden;
  long long N, D, h_ld, V;
  const void* target;
  int target_bytes;
  const float* weight;
  float eps, zeta;
  // of the packed rows
  int* idx;     // [rows_pad] original row
  int* packed;  // [rows_pad] target token
  int* place;   // [N] packed row, or -1
  RowCoef* coef;
  float* zt;
  void* rows;  // [rows_pad, ldc]
  long long ldc, rows_pad;
  int twice;
  // forward
  const float2* parts;
  const float* zsum;
  int tiles;
  float* loss;
  float* lse;
  float* nll;
  // backward
  const float* lse_in;
  const float* nll_in;  // or null
  const float* up;
  long long up_stride;
  // finish
  const float* part32;
  long long ld32;
  int tile_rows, units;  // of its tiles, and how many are worked on at once
  int k_piece;          // stages of K in a piece of the vocabulary
  long long part_room;  // rows that all parts have together
  void* d_hidden;
  long long dh_ld;
};

// The coefficients of a row's gradient (nll: -log p_t, or less than 0: unknown), and an f32 that no |G| exceeds: 0 where
// that is not finite, so that such a row takes no part in the power of two that it shares with others.
__device__ __forceinline__ RowCoef coef_of(const RowArgs& a, float factor, float lse, double nll, unsigned& bound) {
  RowCoef k;
  k.c = lse * LOG2E;
  k.c1 = factor * fmaf(2.0f * a.zeta, lse, 1.0f);
  k.c3 = factor * a.eps / (float)a.V;
  const float c2 = factor * (1.0f - a.eps);
  if (nll < 0.0) {
    k.target = -c2;
  } else {
    const double z2 = 2.0 * a.zeta * lse, eps = a.eps;
    k.target = (float)(factor * ((1.0 + z2) * expm1(-nll) + z2 + eps - eps / (double)a.V));
  }
  const float most = fabsf(k.c1) + fabsf(c2) + fabsf(k.c3);
  bound = isfinite(most) ? __float_as_uint(most) : 0u;
  return k;
}

// Into how many ranges the hidden states' gradient cuts a piece's K.  Its time in stages of a tile (64 of K, 0.28 us):
// whole rounds of tiles over the pairs of SMs, 16 stages to begin and empty a tile, and each part's way out to HBM and
// back.  One thread tries one count.
__device__ __forceinline__ unsigned split_time(const RowArgs& a, int active, int splits, int tile_rows, int units) {
  const long long rows = (active + 255) / 256 * 256, tiles = (active + tile_rows - 1) / tile_rows * ((a.D + BN - 1) / BN);
  if (splits > 1 && (splits * rows > a.part_room || splits * 4 > a.k_piece)) return 0xffffffffu;
  const long long rounds = (tiles * splits + units - 1) / units;
  const float part = (float)active * (float)a.D * 8.0f / 6.5e6f / 0.28f;
  return (unsigned)fminf(4e9f, (float)rounds * (float)((a.k_piece + splits - 1) / splits + 16) + (float)splits * part);
}

// Packed row i: row n, or (n < 0) zeros, behind the rows that count to a whole tile.
__device__ __forceinline__ void put_row(const RowArgs& a, long long i, int active, long long n) {
  uint16_t* to = (uint16_t*)a.rows + i * a.ldc;
  if (n < 0) {
    if (i < (active + 255) / 256 * 256)
      for (long long d = threadIdx.x * 8; d < a.ldc; d += blockDim.x * 8) *(uint4*)(to + d) = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint16_t* from = (const uint16_t*)a.hidden + n * a.h_ld;
  if (((uintptr_t)from & 15) == 0) {
    long long d = threadIdx.x * 8;
    for (; d + 8 <= a.D; d += blockDim.x * 8) *(uint4*)(to + d) = *(const uint4*)(from + d);
    if (d < a.D)
      for (long long e = d; e < a.D; ++e) to[e] = from[e];
  } else {
    for (long long d = threadIdx.x; d < a.D; d += blockDim.x) to[d] = from[d];
  }
}

constexpr int PACK_ROWS = 1024;  // that a block counts through for each row it copies

// Packs the rows that count, in their order (BACKWARD: with their coefficients).  COPY: a block for each packed row,
// which counts for itself and then copies it; the first one writes the rest.  Otherwise one block, and
// lce_gather_kernel copies.
template <bool BACKWARD, bool COPY>
__global__ void __launch_bounds__(PACK_ROWS) lce_pack_kernel(const RowArgs a) {
  depend_wait();
  depend_launch();
  __shared__ int scratch[33], mine;
  __shared__ unsigned most[33];
  const bool writes = !COPY || blockIdx.x == 0;
  // of the rows that count, the one to copy
  const int wanted = !a.twice ? blockIdx.x : blockIdx.x < 2 * TWICE ? blockIdx.x % TWICE : INT_MAX;
  if (threadIdx.x == 0) mine = -1;
  int before = 0;
  unsigned bound = 0;
  for (long long n0 = 0; n0 < a.N; n0 += blockDim.x) {
    const long long n = n0 + threadIdx.x;
    long long t = -1;
    float w = 1.0f;
    if (n < a.N) {
      t = a.target_bytes == 8 ? ((const long long*)a.target)[n] : ((const int*)a.target)[n];
      if (a.weight) w = a.weight[n];
    }
    const bool live = t >= 0 && t < a.V && w != 0.0f;
    int total;
    const int at = before + block_excl_scan_add<int>(live ? 1 : 0, scratch, total);
    if (writes && n < a.N) {
      a.place[n] = live ? at : -1;
      if (!BACKWARD && !live) {
        a.loss[n] = 0.0f;
        if (a.lse) a.lse[n] = 0.0f;
        if (a.nll) a.nll[n] = 0.0f;
      }
    }
    if (live) {
      if (COPY && at == wanted) mine = (int)n;
      if (writes) {
        a.idx[at] = (int)n;
        a.packed[at] = (int)t;
        if (BACKWARD) {
          unsigned most_of;
          a.coef[at] = coef_of(a, w * a.up[n * a.up_stride], a.lse_in[n], a.nll_in ? (double)a.nll_in[n] : -1.0, most_of);
          bound = max(bound, most_of);
        }
      }
    }
    before += total;
  }
  if (COPY) {
    __syncthreads();
    put_row(a, blockIdx.x, before, mine);
  }
  if (!writes) return;
  if (BACKWARD) bound = block_reduce_max<unsigned>(bound, most);
  if (threadIdx.x < 32 && a.part_room) {
    unsigned best = split_time(a, before, threadIdx.x + 1, a.tile_rows, a.units), at = threadIdx.x + 1;
    const unsigned more = split_time(a, before, threadIdx.x + 33, a.tile_rows, a.units);
    if (more < best) {
      best = more;
      at = threadIdx.x + 33;
    }
    const unsigned least = warp_reduce_min<unsigned>(best);
    at = warp_reduce_min<unsigned>(best == least ? at : 1000u);
    if (threadIdx.x == 0) {
      a.plan->splits = (int)at;
      a.plan->part_rows = (before + 255) / 256 * 256;
    }
  }
  if (threadIdx.x == 0) {
    a.plan->active = before;
    a.plan->gmax = bound;
    a.plan->failed = 0;
  }
}

__global__ void __launch_bounds__(256) lce_gather_kernel(const RowArgs a) {
  depend_wait();
  depend_launch();
  const int active = a.plan->active;
  put_row(a, blockIdx.x, active, blockIdx.x < active ? a.idx[blockIdx.x] : -1);
}

// A row's tiles joined: ROWS rows a block (8 share what is read; 1 where there are few).  GRADS: the coefficients of its
// gradient too (up = 1).
template <int ROWS, bool GRADS>
__global__ void __launch_bounds__(256) lce_join_kernel(const RowArgs a) {
  __shared__ float sm[8][ROWS];
  __shared__ double ss[8][ROWS], sz[8][ROWS];
  depend_wait();
  depend_launch();
  const int r = threadIdx.x % ROWS, part = threadIdx.x / ROWS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int active = a.plan->active;
  const long long i = (long long)blockIdx.x * ROWS + r;
  if ((long long)blockIdx.x * ROWS >= active) return;
  float m = -INFINITY;
  double s = 0.0, z = 0.0;
  auto join = [&](float m2, double s2) {
    const float most = fmaxf(m, m2), ref = most == -INFINITY ? 0.0f : most;
    s = s * (double)exp2f(m - ref) + s2 * (double)exp2f(m2 - ref);
    m = most;
  };
  if (i < active) {
    for (int t = part; t < a.tiles; t += 256 / ROWS) {
      const float2 p = a.parts[(long long)t * a.rows_pad + i];
      join(p.x, p.y);
      if (a.zsum) z += a.zsum[(long long)t * a.rows_pad + i];
    }
  }
#pragma unroll
  for (int o = ROWS; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(PESTI_FULL_MASK, m, o);
    const double s2 = __shfl_xor_sync(PESTI_FULL_MASK, s, o);
    z += __shfl_xor_sync(PESTI_FULL_MASK, z, o);
    join(m2, s2);
  }
  if (lane < ROWS) {
    sm[warp][r] = m;
    ss[warp][r] = s;
    sz[warp][r] = z;
  }
  __syncthreads();
  if (threadIdx.x >= ROWS || i >= active) return;
  for (int w = 1; w < 8; ++w) {
    join(sm[w][r], ss[w][r]);
    z += sz[w][r];
  }
  const int n = a.idx[i];
  // log2 of the others' sum, and how far it is above the target's logit
  double zt = a.zt[i];
  if (zt == (double)INFINITY || a.plan->failed) zt = NAN;
  const double rest = (double)m + log2(s), over = rest - zt * (double)LOG2E;
  const double log1p_r = log1p(exp2(-fabs(over)));
  const double nll = over > 0.0 ? over / (double)LOG2E + log1p_r : log1p_r;
  const double lse = over > 0.0 ? rest / (double)LOG2E + log1p_r : zt + nll, eps = a.eps;
  const float w = a.weight ? a.weight[n] : 1.0f;
  double loss = (1.0 - eps) * nll + (double)a.zeta * lse * lse;
  if (a.eps != 0.0f) loss += eps * (lse - z / (double)a.V);
  a.loss[n] = (float)(w * loss);
  if (a.lse) a.lse[n] = (float)lse;
  if (a.nll) a.nll[n] = (float)nll;
  if (GRADS) {
    unsigned bound;
    a.coef[i] = coef_of(a, w, (float)lse, nll, bound);
    atomicMax(&a.plan->gmax, bound);
  }
}

// The hidden states' gradient: the parts summed in their order, to the rows' own places; padded rows get zeros.  Four
// columns a thread, eight parts at a time in flight.  TEAMS 8: a block has 128 columns of a row, and eight teams an
// eighth of the parts each (few rows: 37 rows of 64 parts took 28 us in one team, 11 in eight); TEAMS 1: 1024 columns.
template <bool BF16, int TEAMS>
__global__ void __launch_bounds__(256) lce_finish_kernel(const RowArgs a) {
  depend_wait();
  depend_launch();
  constexpr int THREADS = 256 / TEAMS;
  __shared__ float4 sums[TEAMS > 1 ? TEAMS : 1][THREADS];
  const long long n = blockIdx.y;
  const int i = a.place[n], splits = a.plan->splits, at = threadIdx.x % THREADS, team = threadIdx.x / THREADS;
  const long long part = (long long)a.plan->part_rows * a.ld32, d = ((long long)blockIdx.x * THREADS + at) * 4;
  const float* from = a.part32 + (long long)max(i, 0) * a.ld32 + d;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](float4 x) {
    v.x += x.x;
    v.y += x.y;
    v.z += x.z;
    v.w += x.w;
  };
  if (i >= 0 && d < a.D) {  // (columns of a part are padded to four)
    const int s1 = splits * (team + 1) / TEAMS;
#pragma unroll 8
    for (int s = splits * team / TEAMS; s < s1; ++s) add(__ldcs((const float4*)(from + s * part)));
    if (a.twice) {
#pragma unroll 8
      for (int s = splits * team / TEAMS; s < s1; ++s) add(__ldcs((const float4*)(from + s * part + TWICE * a.ld32)));
    }
  }
  if (TEAMS > 1) {
    sums[team][at] = v;
    __syncthreads();
    if (team) return;
    for (int k = 1; k < TEAMS; ++k) add(sums[k][at]);
  }
  if (d >= a.D) return;
  // (a wait that gave up makes NaN, in padded rows too)
  const float scale = a.plan->failed ? NAN : pow2(-grad_shift<BF16>(a.plan));
  const uint2 w = make_uint2(pack2<BF16>(v.x * scale, v.y * scale), pack2<BF16>(v.z * scale, v.w * scale));
  uint16_t* to = (uint16_t*)a.d_hidden + n * a.dh_ld + d;
  if (((uintptr_t)to & 7) == 0 && d + 4 <= a.D) {
    *(uint2*)to = w;
  } else {
    const uint16_t h[4] = {(uint16_t)w.x, (uint16_t)(w.x >> 16), (uint16_t)w.y, (uint16_t)(w.y >> 16)};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d + j < a.D) to[j] = h[j];
  }
}

}  // namespace pesti_lce
