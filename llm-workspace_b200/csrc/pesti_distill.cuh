// Distillation from a teacher's top logits: loss and gradient over rows of
// student logits.
//
// For one row, z = x/T over V tokens, p = softmax(z); the teacher lists k
// entries (i_j, t_j):
//   no log sum:   q_j = exp(t_j/T) / sum_j exp(t_j/T),  q_t = 0
//   log sum L:    q_j = exp(t_j/T - L),  q_t = max(0, 1 - sum_j q_j)
// With p_t the mass of the tokens that are not listed (q_t counts as 0 where
// p_t is 0 in 64 bits), Q = sum_j q_j, and w the row's weight:
//   loss     = w T^2 [ sum_j q_j (log q_j - log p_{i_j}) + q_t (log q_t - log p_t) ]
//   grad_v   = w T [ (Q + q_t) p_v - sum_{j: i_j = v} q_j ]          v listed
//            = w T [ (Q + q_t) - q_t / p_t ] p_v                     else
// So outside the list the gradient is one factor of the row times 2^(x*C - R),
// C = log2(e)/T; the k listed places are written apart.
//
// distill_row_kernel: a cluster of CTAs per row.  A row's units
//   (pesti_rowscan.cuh) are split over the cluster and streamed once; with a
//   gradient they stay in shared memory until the row's sum is known, so the
//   logits cross HBM once.  p_t is summed from the unlisted tokens themselves:
//   1 - sum p would lose it when the list holds nearly all the mass.  One warp
//   of each CTA works on the list meanwhile.
// distill_backward_kernel: the gradient alone, from what the forward pass kept
//   of each row (8 numbers).
//
// Sums: 64 terms of a lane and unit in f32, units, lanes, warps and CTAs in
// 64 bits in a fixed order.  Everything of the list (k <= 256 entries) is in
// 64 bits: the loss is a difference of nearly equal logarithms.
#pragma once
#include "pesti_common.cuh"
#include "pesti_rowscan.cuh"

namespace pesti_rows {

constexpr int MAX_TOP = 256;
constexpr int HASH = 512;
constexpr int ROW_WARPS = 15;                         // streaming warps
constexpr int ROW_THREADS = (ROW_WARPS + 1) * 32;     // and the list's
constexpr int MAX_CLUSTER = 16;
constexpr int STATS = 8;
constexpr double ONE_LN2 = 0.69314718055994530942;

// Numbers of a row that the backward pass needs.
enum { ST_MS = 0, ST_A = 1, ST_LOGQ = 2, ST_TOTAL = 3, ST_MALL = 4, ST_LOGS = 5 };

struct DistillArgs {
  const void* logits;
  long long ld, V;
  const int32_t* idx;
  const void* val;
  long long idx_ld, val_ld;
  int val_dtype;  // 0 f32, 1 bf16, 2 f16
  int k;
  const float* teacher_lse;
  const float* weight;
  double T;
  double C;       // log2(e) / T
  float c, c_lo;  // C = c + c_lo, c_lo >= 0
  float* loss;
  double* stats;
  void* grad;
  long long grad_ld;
  long long units, per_cta;
  int keep;       // the CTA's units stay in shared memory
  const float* up;
  long long up_stride;
};

__device__ __forceinline__ double teacher_value(const DistillArgs& a, long long n, int j) {
  const long long at = n * a.val_ld + j;
  if (a.val_dtype == 0) return (double)((const float*)a.val)[at];
  if (a.val_dtype == 1) return (double)__bfloat162float(((const __nv_bfloat16*)a.val)[at]);
  return (double)__half2float(((const __half*)a.val)[at]);
}

// e = 2^(x*C - R) relative to the reference of m, in 64 bits.
__device__ __forceinline__ double exact_term(float x, float m, const DistillArgs& a) {
  if (x != x) return (double)x;
  if (m == neg_inf()) return 0.0;
  if (is_far(m, a.c)) return x == m ? 1.0 : 0.0;
  return exp2((double)x * a.C - (double)ceilf(m * a.c));
}

// The reference R of a row's or unit's largest logit m (0 where it is not used).
__device__ __forceinline__ float reference(float m, float c) {
  return m > neg_inf() && !is_far(m, c) ? ceilf(m * c) : 0.0f;
}

// A term where m is far: 1 at m itself.
__device__ __forceinline__ float far_term(float x, float m) { return x == m ? 1.0f : x != x ? x : 0.0f; }

// Sum of a lane's terms of a unit.
template <typename T>
__device__ __forceinline__ float sum_terms(const uint4 (&v)[UNIT_VECS], float m, const DistillArgs& a) {
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
  if (m > neg_inf() && is_far(m, a.c)) {
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i)
#pragma unroll
      for (int q = 0; q < Elem<T>::PAIRS; ++q) {
        const float2 x = Elem<T>::pair(v[i], q);
        s0 = add2(s0, make_float2(far_term(x.x, m), far_term(x.y, m)));
      }
  } else {
    const float R = reference(m, a.c);
    const float2 c2 = make_float2(a.c, a.c), lo2 = make_float2(a.c_lo, a.c_lo), r2 = make_float2(-R, -R);
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i)
#pragma unroll
      for (int q = 0; q < Elem<T>::PAIRS; ++q) {
        const float2 x = Elem<T>::pair(v[i], q);
        const float2 t = fma2(x, lo2, fma2(x, c2, r2));
        const float2 e = make_float2(ex2(t.x), ex2(t.y));
        if (q & 1)
          s1 = add2(s1, e);
        else
          s0 = add2(s0, e);
      }
  }
  return (s0.x + s0.y) + (s1.x + s1.y);
}

struct Partial {
  float m;
  double s;
};

// Joins one partial sum per lane; NaN stays NaN (a scale multiplies it).
__device__ __forceinline__ Partial warp_join(Partial p, float c) {
  const float m = warp_max(p.m);
  p.s = warp_reduce_add(p.s * ref_scale(p.m, m, c));
  p.m = m;
  return p;
}

struct RowShared {
  int32_t idx[MAX_TOP];   // -1: no entry
  int32_t hash[HASH];
  float x[MAX_TOP];       // the places' logits
  double q[MAX_TOP];
  double qs[MAX_TOP];     // sum of q over equal tokens
  double e[MAX_TOP];      // 2^(x C - R) for the largest listed logit's R
  uint8_t first[MAX_TOP]; // first entry of its token
  Partial warp[ROW_WARPS];
  Partial cta;
  double total, e_scale;  // Q + q_t; factor from e to p
  float m_s, A;
};

// What the list's warp knows before the row's sum (the same in every lane).
struct ListPart {
  double Q, norm, rest;  // sum of q, log of the teacher's normaliser, max(0, 1 - Q) or 0
  Partial member;        // listed tokens, each once
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ Partial peer_partial(const Partial* p, uint32_t rank) {
  const uint32_t local = (uint32_t)__cvta_generic_to_shared(p);
  uint32_t at;
  Partial r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r.m) : "r"(at) : "memory");
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(r.s) : "r"(at + 8) : "memory");
  return r;
}

// Sets listed elements of the unit to -inf in the lanes' registers.
template <typename T>
__device__ __forceinline__ void leave_out(uint4 (&v)[UNIT_VECS], const int32_t* idx, int k, long long first, int lane) {
  constexpr int VE = Elem<T>::VE;
  for (int j0 = 0; j0 < k; j0 += 32) {
    const int j = j0 + lane;
    const long long o = j < k && idx[j] >= 0 ? (long long)idx[j] - first : -1;
    uint32_t in = __ballot_sync(FULL, o >= 0 && o < UNIT_SLOTS * VE);
    while (in) {
      const int from = __ffs(in) - 1;
      in &= in - 1;
      const int e = __shfl_sync(FULL, (int)o, from);
      const int slot = e / VE, sub = e % VE;
      if (lane == (slot & 31)) {
#pragma unroll
        for (int i = 0; i < UNIT_VECS; ++i)
          if (i == (slot >> 5)) Elem<T>::put(v[i], sub, Elem<T>::NEG_INF);
      }
    }
  }
}

// Gradient of one vector (slot of the aligned address space) of a row.
template <typename T>
__device__ __forceinline__ void store_vec(T* grow, long long lo, long long V, bool vec, const uint4& g) {
  if (vec && lo >= 0 && lo + Elem<T>::VE <= V) {
    *(uint4*)(grow + lo) = g;
  } else {
#pragma unroll
    for (int q = 0; q < Elem<T>::PAIRS; ++q) {
      const float2 f = Elem<T>::pair(g, q);
      const long long i = lo + 2 * q;
      if (i >= 0 && i < V) Elem<T>::store(grow, i, f.x);
      if (i + 1 >= 0 && i + 1 < V) Elem<T>::store(grow, i + 1, f.y);
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 grad_vec(const uint4& v, float2 c2, float2 lo2, float2 r2, float A) {
  uint4 g;
#pragma unroll
  for (int q = 0; q < Elem<T>::PAIRS; ++q) {
    const float2 x = Elem<T>::pair(v, q);
    const float2 t = fma2(x, lo2, fma2(x, c2, r2));
    Elem<T>::pack(g, q, make_float2(ex2(t.x) * A, ex2(t.y) * A));
  }
  return g;
}

// The gradient of a unit outside the list: A times the terms.
template <typename T>
__device__ __forceinline__ void store_unit(T* grow, const uint4 (&v)[UNIT_VECS], int head, long long V, bool vec,
                                           long long u, int lane, float m, float A, const DistillArgs& a) {
  constexpr int VE = Elem<T>::VE;
  const long long first = (u * UNIT_SLOTS + lane) * VE - head;
  if (m > neg_inf() && is_far(m, a.c)) {
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i) {
      uint4 g;
#pragma unroll
      for (int q = 0; q < Elem<T>::PAIRS; ++q) {
        const float2 x = Elem<T>::pair(v[i], q);
        Elem<T>::pack(g, q, make_float2(far_term(x.x, m) * A, far_term(x.y, m) * A));
      }
      store_vec<T>(grow, first + i * 32 * VE, V, vec, g);
    }
  } else {
    const float R = reference(m, a.c);
    const float2 c2 = make_float2(a.c, a.c), lo2 = make_float2(a.c_lo, a.c_lo), r2 = make_float2(-R, -R);
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i)
      store_vec<T>(grow, first + i * 32 * VE, V, vec, grad_vec<T>(v[i], c2, lo2, r2, A));
  }
}

// Zeros for units [ua, ub) of a gradient row.
template <typename T>
__device__ __forceinline__ void zero_units(T* grow, int head, long long V, bool vec, long long ua, long long ub) {
  const uint4 z = make_uint4(0, 0, 0, 0);
  for (long long s = ua * UNIT_SLOTS + threadIdx.x; s < ub * UNIT_SLOTS; s += blockDim.x)
    store_vec<T>(grow, s * Elem<T>::VE - head, V, vec, z);
}

// The list's warp: teacher probabilities, equal tokens, and the listed tokens' terms.
__device__ __forceinline__ ListPart list_part(RowShared& sh, const DistillArgs& a, long long n, int lane) {
  const double inf = (double)pos_inf();
  ListPart r;
  double mt = -inf;
  float mx = neg_inf();
  for (int i = lane; i < HASH; i += 32) sh.hash[i] = -1;
  for (int j = lane; j < a.k; j += 32) {
    const bool in = sh.idx[j] >= 0;
    const double t = in ? teacher_value(a, n, j) / a.T : -inf;
    sh.q[j] = t;
    mt = !(t <= mt) ? t : mt;  // NaN is taken over
    if (in) mx = fmaxf(mx, sh.x[j]);
  }
  mx = warp_max(mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double y = __shfl_xor_sync(FULL, mt, o);
    mt = mt != mt ? mt : !(y <= mt) ? y : mt;
  }
  if (a.teacher_lse) {
    r.norm = (double)a.teacher_lse[n];
  } else {
    r.norm = 0.0;
    if (mt != -inf) {
      double z = 0.0;
      for (int j = lane; j < a.k; j += 32) z += exp(sh.q[j] - mt);
      r.norm = mt + log(warp_reduce_add(z));
    }
  }
  r.Q = 0.0;
  bool dup = false;
  for (int j = lane; j < a.k; j += 32) {
    const int32_t id = sh.idx[j];
    const double q = id >= 0 ? exp(sh.q[j] - r.norm) : 0.0;
    sh.q[j] = q;
    sh.qs[j] = q;
    sh.first[j] = id >= 0;
    sh.e[j] = id >= 0 ? exact_term(sh.x[j], mx, a) : 0.0;
    r.Q += q;
    if (id >= 0) {
      uint32_t h = ((uint32_t)id * 2654435761u) >> 23;
      for (;;) {
        const int32_t had = atomicCAS(&sh.hash[h], -1, id);
        if (had == -1) break;
        if (had == id) {
          dup = true;
          break;
        }
        h = (h + 1) & (HASH - 1);
      }
    }
  }
  r.Q = warp_reduce_add(r.Q);
  if (__any_sync(FULL, dup)) {
    // a token listed twice: the first entry stands for it
    __syncwarp();
    for (int j = lane; j < a.k; j += 32)
      if (sh.idx[j] >= 0) {
        double s = 0.0;
        bool first = true;
        for (int o = 0; o < a.k; ++o)
          if (sh.idx[o] == sh.idx[j]) {
            s += sh.q[o];
            first = first && o >= j;
          }
        sh.qs[j] = s;
        sh.first[j] = first;
      }
  }
  __syncwarp();
  r.member.m = mx;
  r.member.s = 0.0;
  for (int j = lane; j < a.k; j += 32)
    if (sh.first[j]) r.member.s += sh.e[j];
  r.member.s = warp_reduce_add(r.member.s);
  const double rest = 1.0 - r.Q;
  r.rest = a.teacher_lse ? (rest < 0.0 ? 0.0 : rest) : 0.0;
  return r;
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(ROW_THREADS, 2) distill_row_kernel(const __grid_constant__ DistillArgs a) {
  extern __shared__ uint4 kept[];
  __shared__ RowShared sh;
  constexpr int VE = Elem<T>::VE;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const uint32_t csize = cluster_size(), crank = cluster_rank();
  const long long n = blockIdx.x / csize;
  const T* row = (const T*)a.logits + n * a.ld;
  const int head = row_head<T>(row);
  const long long ua = min(a.units, (long long)crank * a.per_cta), ub = min(a.units, ua + a.per_cta);
  T* grow = GRAD ? (T*)a.grad + n * a.grad_ld : nullptr;
  const bool vec = GRAD && row_head<T>(grow) == head;
  const float w = a.weight ? a.weight[n] : 1.0f;
  if (w == 0.0f) {
    // the row is not read (every CTA of the cluster is here)
    if (GRAD) zero_units<T>(grow, head, a.V, vec, ua, ub);
    if (crank == 0 && tid == 0) a.loss[n] = 0.0f;
    return;
  }
  const bool tail = a.teacher_lse != nullptr;
  ListPart list;
  if (wid == ROW_WARPS) {
    for (int j = lane; j < a.k; j += 32) {
      const int32_t id = a.idx[n * a.idx_ld + j];
      const bool in = id >= 0 && id < a.V;
      sh.idx[j] = in ? id : -1;
      sh.x[j] = in ? Elem<T>::load(row, id) : neg_inf();
    }
    __syncthreads();
    list = list_part(sh, a, n, lane);
  } else {
    Partial acc{neg_inf(), 0.0};
    uint4 v[UNIT_VECS];
    long long u = ua + wid;
    if (u < ub) load_unit<T, !GRAD>(v, row, head, a.V, u, lane);
    __syncthreads();  // the list is there
    while (u < ub) {
      if (GRAD && a.keep) {
#pragma unroll
        for (int i = 0; i < UNIT_VECS; ++i) kept[(u - ua) * UNIT_SLOTS + i * 32 + lane] = v[i];
      }
      if (tail) leave_out<T>(v, sh.idx, a.k, u * UNIT_SLOTS * VE - head, lane);
      float m = neg_inf();
#pragma unroll
      for (int i = 0; i < UNIT_VECS; ++i) m = fmaxf(m, Elem<T>::vec_max(v[i]));
      m = fmaxf(acc.m, warp_max(m));
      acc.s = acc.s * ref_scale(acc.m, m, a.c) + (double)sum_terms<T>(v, m, a);
      acc.m = m;
      u += ROW_WARPS;
      if (u < ub) load_unit<T, !GRAD>(v, row, head, a.V, u, lane);
    }
    acc.s = warp_reduce_add(acc.s);  // every lane has the same reference
    if (lane == 0) sh.warp[wid] = acc;
  }
  __syncthreads();
  Partial s{neg_inf(), 0.0};
  if (wid == ROW_WARPS) {
    if (lane < ROW_WARPS) s = sh.warp[lane];
    s = warp_join(s, a.c);
    if (lane == 0) sh.cta = s;
  }
  if (csize > 1) {
    cluster_arrive();
    cluster_wait();
  }
  // the list's warp of every CTA puts the row together
  const double pos = (double)pos_inf();
  float m_all = neg_inf();
  double S = 0.0, scale = 1.0, total = 0.0, q_t = 0.0, A = 0.0;
  if (wid == ROW_WARPS) {
    if (csize > 1) {
      s = Partial{neg_inf(), 0.0};
      if (lane < csize) s = peer_partial(&sh.cta, lane);
      s = warp_join(s, a.c);
    }
    // all tokens: what was streamed, and the listed ones where they were left out
    m_all = tail ? fmaxf(s.m, list.member.m) : s.m;
    scale = ref_scale(s.m, m_all, a.c);
    const double e_scale = ref_scale(list.member.m, m_all, a.c);
    S = s.s * scale + (tail ? list.member.s * e_scale : 0.0);
    if (m_all == pos_inf()) S = pos - pos;  // +inf logits have no softmax: NaN
    q_t = list.rest;
    if (s.s == 0.0 || scale == 0.0) q_t = q_t == q_t ? 0.0 : q_t;  // no unlisted token with a probability (in 64 bits)
    total = list.Q + q_t;
    // outside the list: grad = A * 2^(x C - Rs)
    A = S;
    if (S == S) A = s.s > 0.0 ? a.T * (total * scale / S - (q_t != 0.0 ? q_t / s.s : 0.0)) : 0.0;
    if (lane == 0) {
      sh.A = (float)(A * (double)w);
      sh.total = total;
      // p of a listed token; a row of -inf alone has none
      sh.e_scale = S == 0.0 ? 0.0 : e_scale / S;
      sh.m_s = s.m;
    }
  }
  if (csize > 1) cluster_arrive();  // done with the others' shared memory
  if (GRAD) __syncthreads();
  if (wid == ROW_WARPS) {
    if (crank == 0) {
      const bool none = !(m_all > neg_inf()) && S == S;  // every logit is -inf
      const bool far = !none && is_far(m_all, a.c);
      // log sum exp((x - m_all)/T)
      const double logS = none ? 0.0 : far ? log(S) : ONE_LN2 * (log2(S) - ((double)m_all * a.C - (double)reference(m_all, a.c)));
      double l = 0.0;
      for (int j = lane; j < a.k; j += 32) {
        const double q = sh.q[j];
        if (sh.idx[j] >= 0 && q != 0.0) {
          const double x = (double)sh.x[j];
          const double logp = none || x == -pos ? (S == S ? -pos : S) : (x - (double)m_all) / a.T - logS;
          l += q * ((teacher_value(a, n, j) / a.T - list.norm) - logp);
        }
      }
      l = warp_reduce_add(l);
      // p_t = s.s * scale / S
      if (q_t != 0.0) l += q_t * (log(q_t) - (log(s.s) + log(scale) - log(S)));
      if (S != S) l = S;
      if (lane == 0) {
        a.loss[n] = (float)((double)w * a.T * a.T * l);
        if (a.stats) {
          double* st = a.stats + n * STATS;
          st[ST_MS] = (double)s.m;
          st[ST_A] = A;
          st[ST_LOGQ] = list.norm;
          st[ST_TOTAL] = total;
          st[ST_MALL] = (double)m_all;
          st[ST_LOGS] = logS;
        }
      }
    }
  } else if (GRAD) {
    const float m = sh.m_s, f = sh.A;
    for (long long u = ua + wid; u < ub; u += ROW_WARPS) {
      uint4 v[UNIT_VECS];
      if (a.keep) {
#pragma unroll
        for (int i = 0; i < UNIT_VECS; ++i) v[i] = kept[(u - ua) * UNIT_SLOTS + i * 32 + lane];
      } else {
        load_unit<T, false>(v, row, head, a.V, u, lane);
      }
      store_unit<T>(grow, v, head, a.V, vec, u, lane, m, f, a);
    }
  }
  if (GRAD) {
    __syncthreads();
    // the listed places of this CTA's part
    const long long from = ua * UNIT_SLOTS * VE - head, to = ub * UNIT_SLOTS * VE - head;
    for (int j = tid; j < a.k; j += ROW_THREADS) {
      const long long id = sh.idx[j];
      if (id >= 0 && sh.first[j] && id >= from && id < to)
        Elem<T>::store(grow, id, (float)((double)w * a.T * (sh.total * (sh.e[j] * sh.e_scale) - sh.qs[j])));
    }
  }
  if (csize > 1) cluster_wait();
}

constexpr int BACK_WARPS = 8;

// One warp per unit of a row, BACK_WARPS units per block.
template <typename T>
__global__ void __launch_bounds__(BACK_WARPS * 32) distill_backward_kernel(const __grid_constant__ DistillArgs a,
                                                                           long long blocks_per_row) {
  __shared__ int32_t in_idx[MAX_TOP], in_j[MAX_TOP];
  __shared__ float in_x[MAX_TOP];
  __shared__ double in_q[MAX_TOP];
  __shared__ int count;
  constexpr int VE = Elem<T>::VE;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const long long n = blockIdx.x / blocks_per_row;
  const long long ua = (blockIdx.x - n * blocks_per_row) * BACK_WARPS, ub = min(a.units, ua + BACK_WARPS);
  const T* row = (const T*)a.logits + n * a.ld;
  T* grow = (T*)a.grad + n * a.grad_ld;
  const int head = row_head<T>(row);
  const bool vec = row_head<T>(grow) == head;
  const float w = a.weight ? a.weight[n] : 1.0f;
  if (w == 0.0f) {
    zero_units<T>(grow, head, a.V, vec, ua, ub);
    return;
  }
  if (tid == 0) count = 0;
  __syncthreads();
  const double* st = a.stats + n * STATS;
  const double scale = (double)w * (double)a.up[n * a.up_stride];
  const long long u = ua + wid;
  uint4 v[UNIT_VECS];
  if (u < ub) load_unit<T, false>(v, row, head, a.V, u, lane);
  // the list's places in this block's part, read before anything is written
  const long long from = ua * UNIT_SLOTS * VE - head, to = ub * UNIT_SLOTS * VE - head;
  if (tid < a.k) {
    const long long id = a.idx[n * a.idx_ld + tid];
    if (id >= 0 && id < a.V && id >= from && id < to) {
      const int at = atomicAdd(&count, 1);
      in_idx[at] = (int32_t)id;
      in_j[at] = tid;
      in_x[at] = Elem<T>::load(row, id);
      in_q[at] = exp(teacher_value(a, n, tid) / a.T - st[ST_LOGQ]);
    }
  }
  const float m = (float)st[ST_MS], A = (float)(st[ST_A] * scale);
  __syncthreads();
  if (u < ub) store_unit<T>(grow, v, head, a.V, vec, u, lane, m, A, a);
  __syncthreads();
  const int cnt = count;
  for (int i = tid; i < cnt; i += BACK_WARPS * 32) {
    // entries of the same token add up in the list's order; the first one writes
    bool first = true;
    double qs = 0.0;
    for (int last = -1;;) {
      int next = MAX_TOP, at = -1;
      for (int o = 0; o < cnt; ++o)
        if (in_idx[o] == in_idx[i] && in_j[o] > last && in_j[o] < next) {
          next = in_j[o];
          at = o;
        }
      if (at < 0) break;
      if (next < in_j[i]) first = false;
      qs += in_q[at];
      last = next;
    }
    if (first) {
      const double x = (double)in_x[i], logs = st[ST_LOGS];
      const double p = x == -(double)pos_inf() && logs == logs ? 0.0 : exp((x - st[ST_MALL]) / a.T - logs);
      Elem<T>::store(grow, in_idx[i], (float)(scale * a.T * (st[ST_TOTAL] * p - qs)));
    }
  }
}

}  // namespace pesti_rows
