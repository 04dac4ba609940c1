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
// distill_row_kernel: clusters of CTAs that walk over rows.  A row's segments
//   (pesti_rowscan.cuh) are split over the cluster's streaming warps.  Each
//   lane copies its own 16-byte vectors into slots of its own in shared memory
//   (cp.async), several batches ahead and over the row's end into the next
//   row, so the copies never pause for what a row costs besides its data.
//   With a gradient the slots hold the row's part until its sum is known (the
//   logits cross HBM once) and each is refilled for the next row once its
//   gradient is written.  One warp works on the next row's list, one joins
//   the sums, passes them on in the cluster and finishes the row.  (No register
//   may spill: next to 200 KB of shared memory there is no L1 to speak of.)
//   p_t is summed from the unlisted tokens themselves: 1 - sum p would lose it
//   when the list holds nearly all the mass.
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
constexpr int ROW_WARPS = 12;                         // streaming warps
constexpr int JOIN_WARP = ROW_WARPS;
constexpr int ROW_THREADS = (ROW_WARPS + 2) * 32;     // the list warp behind it
constexpr int MAX_CLUSTER = 16;
constexpr int BATCH = 4;                              // segments that a warp takes at a time
constexpr int MAX_KEEP = 15;                          // segments of a warp that stay: two CTAs fit an SM
constexpr int WAIT_LIMIT = 1 << 20;
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
  long long units;          // backward: units of a row
  long long N;              // rows
  int warp_segs;            // segments of a warp's part of a row
  int batches;              // in batches of BATCH
  int slots, ring_segs;     // slots and segments of a warp's ring
  int keep;                 // a slot for every batch: they stay until the gradient is written
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

// Sum of a lane's terms.
template <typename T, int NV>
__device__ __forceinline__ float sum_terms(const uint4 (&v)[NV], float m, const DistillArgs& a) {
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
  if (m > neg_inf() && is_far(m, a.c)) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int q = 0; q < Elem<T>::PAIRS; ++q) {
        const float2 x = Elem<T>::pair(v[i], q);
        s0 = add2(s0, make_float2(far_term(x.x, m), far_term(x.y, m)));
      }
  } else {
    const float R = reference(m, a.c);
    const float2 c2 = make_float2(a.c, a.c), lo2 = make_float2(a.c_lo, a.c_lo), r2 = make_float2(-R, -R);
#pragma unroll
    for (int i = 0; i < NV; ++i)
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

// One row's list.
struct ListBuf {
  int32_t idx[MAX_TOP];  // -1: no entry
  float x[MAX_TOP];      // the places' logits
  double q[MAX_TOP];
  union {
    double qs[MAX_TOP];  // sum of q over equal tokens
    int32_t hash[HASH];  // while equal tokens are looked for
  };
  double e[MAX_TOP];       // 2^(x C - R) for the largest listed logit's R
  uint8_t first[MAX_TOP];  // first entry of its token
  double Q, norm, rest;    // sum of q, log of the teacher's normaliser, max(0, 1 - Q) or 0
  Partial member;          // listed tokens, each once
};

struct RowShared {
  ListBuf list[2];
  Partial warp[2][ROW_WARPS];   // by row parity
  Partial cta[2][MAX_CLUSTER];  // the cluster's sums
  unsigned long long arrived[2];
  float m_s, A;  // of the row whose gradient is written
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

// Named barriers (0 is __syncthreads).  By row parity: the list is there, the list is free, the warps' sums are there; then: the row is known, its part is written.
enum { BAR_FULL = 1, BAR_EMPTY = 3, BAR_SUMS = 5, BAR_ROW = 7, BAR_DONE = 8 };
__device__ __forceinline__ void bar_sync(int id, int threads) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  __syncwarp();
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Puts a partial sum into CTA `rank`'s shared memory and signs in there.
__device__ __forceinline__ void send_partial(Partial* to, unsigned long long* bar, uint32_t rank, const Partial& p) {
  uint32_t at, b;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(to)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(p.m) : "memory");
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at + 8), "d"(p.s) : "memory");
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(b) : "memory");
}
// False if the others have not signed in within the limit.
__device__ __forceinline__ bool wait_partials(unsigned long long* bar, uint32_t parity) {
  const uint32_t b = (uint32_t)__cvta_generic_to_shared(bar);
  for (int i = 0; i < WAIT_LIMIT; ++i) {
    uint32_t ok;
    asm volatile(
        "{.reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;}"
        : "=r"(ok)
        : "r"(b), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}

__device__ __forceinline__ void copy_vec(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most n of the lane's latest groups are in flight.
__device__ __forceinline__ void copies_wait(int n) {
  if (n <= 0)
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (n == 1)
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (n == 2)
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  else
    asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// The rows of a cluster, rows of weight 0 left out: every warp walks over them by itself.
struct RowWalk {
  int first, step, at;  // rows first + i * step < N; window of 32 at i = `at`
  uint32_t left;

  __device__ __forceinline__ RowWalk(int cluster, int clusters) : first(cluster), step(clusters), at(-32), left(0u) {}
  // The next row, or -1.  `skipped` is called with each row of weight 0 that is passed.
  template <typename F>
  __device__ __forceinline__ int next(const DistillArgs& a, F skipped) {
    while (left == 0u) {
      at += 32;
      const long long i = first + (long long)(at + (int)(threadIdx.x & 31)) * step;
      const bool in = i < a.N;
      const bool none = in && a.weight && a.weight[i] == 0.0f;
      left = __ballot_sync(FULL, in && !none);
      uint32_t zero = __ballot_sync(FULL, none);
      if ((left | zero) == 0u) return -1;
      for (; zero; zero &= zero - 1) skipped(first + (at + __ffs(zero) - 1) * step);
    }
    const int i = at + __ffs(left) - 1;
    left &= left - 1;
    return first + i * step;
  }
};

// A warp's part of a row, for one lane.  Offsets within a row fit 32 bits (V <= 2^30).
template <typename T>
struct Part {
  static constexpr int VE = Elem<T>::VE, SEG = 32 * VE;
  const T* row;
  int lo;       // element of the lane's first vector
  int segs;     // segments of the part
  bool inside;  // every vector lies in the row

  __device__ __forceinline__ Part(const DistillArgs& a, int n, int part, int lane) {
    row = (const T*)a.logits + (long long)n * a.ld;
    const int head = row_head<T>(row), V = (int)a.V;
    const int first = part * a.warp_segs;
    segs = max(0, min(a.warp_segs, (head + V + SEG - 1) / SEG - first));
    const int from = first * SEG - head;
    inside = from >= 0 && from + segs * SEG <= V;
    lo = from + lane * VE;
  }
  __device__ __forceinline__ int count(int b) const {
    return max(0, min(BATCH, segs - b * BATCH));
  }
  __device__ __forceinline__ bool whole(const DistillArgs& a, int at) const { return at >= 0 && at + VE <= (int)a.V; }
  // Starts the copies of batch b into the lane's slot (one group, empty if there are none).
  __device__ __forceinline__ void copy(const DistillArgs& a, int b, uint32_t slot) const {
    const int n = count(b), at = lo + b * BATCH * SEG;
    const T* from = row + at;
    if (inside && n == BATCH) {
#pragma unroll
      for (int i = 0; i < BATCH; ++i) copy_vec(slot + i * 512, from + i * SEG);
    } else {
      for (int i = 0; i < n; ++i)
        if (whole(a, at + i * SEG)) copy_vec(slot + i * 512, from + i * SEG);
    }
    copies_commit();
  }
  // Completes what copy() brought: the row's ragged ends, and -inf behind them.
  __device__ __forceinline__ void settle(const DistillArgs& a, int b, uint4* slot) const {
    if (inside) return;
    const int n = count(b), at = lo + b * BATCH * SEG;
    for (int i = 0; i < n; ++i)
      if (!whole(a, at + i * SEG)) slot[i * 32] = load_edge<T>(row, at + i * SEG, a.V);
  }
  // Sets listed elements to -inf in the lanes' slots (their gradients are written apart).
  __device__ __forceinline__ void leave_out(const DistillArgs& a, int b, const int32_t* idx, uint4* slot, int lane) const {
    const int from = lo - lane * VE + b * BATCH * SEG, n = count(b) * SEG;
    for (int j0 = 0; j0 < a.k; j0 += 32) {
      const int j = j0 + lane, id = j < a.k ? idx[j] : -1;
      uint32_t in = __ballot_sync(FULL, id >= 0 && (uint32_t)(id - from) < (uint32_t)n);
      while (in) {
        const int e = __shfl_sync(FULL, id, __ffs(in) - 1) - from;
        in &= in - 1;
        if (lane == ((e / VE) & 31)) Elem<T>::store(slot + e / SEG * 32, e % VE, neg_inf());
      }
    }
  }
};

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

// 16-bit gradients leave x*c_lo out but for its value at m, which goes into A (near_factor): the rest,
// |(x - m) c_lo| < 2^-24 |(x - m) C|, is far below their rounding.
template <typename T>
__device__ __forceinline__ float near_factor(float A, float m, const DistillArgs& a) {
  return sizeof(T) == 2 && m > neg_inf() && !is_far(m, a.c) ? A * ex2(m * a.c_lo) : A;
}
template <typename T>
__device__ __forceinline__ uint4 grad_vec(const uint4& v, float2 c2, float2 lo2, float2 r2, float A) {
  const float2 A2 = make_float2(A, A);
  uint4 g;
#pragma unroll
  for (int q = 0; q < Elem<T>::PAIRS; ++q) {
    const float2 x = Elem<T>::pair(v, q);
    float2 t = fma2(x, c2, r2);
    if (sizeof(T) == 4) t = fma2(x, lo2, t);
    Elem<T>::pack(g, q, mul2(make_float2(ex2(t.x), ex2(t.y)), A2));
  }
  return g;
}

// The gradient outside the list of a vector that may reach over the row's ends, or whose logits are far.
template <typename T>
__device__ __forceinline__ void store_any(T* grow, const uint4& v, long long lo, long long V, float m, float A,
                                          const DistillArgs& a) {
  uint4 g;
  if (m > neg_inf() && is_far(m, a.c)) {
#pragma unroll
    for (int q = 0; q < Elem<T>::PAIRS; ++q) {
      const float2 x = Elem<T>::pair(v, q);
      Elem<T>::pack(g, q, make_float2(far_term(x.x, m) * A, far_term(x.y, m) * A));
    }
  } else {
    const float R = reference(m, a.c);
    g = grad_vec<T>(v, make_float2(a.c, a.c), make_float2(a.c_lo, a.c_lo), make_float2(-R, -R),
                    near_factor<T>(A, m, a));
  }
  store_vec<T>(grow, lo, V, row_head<T>(grow + lo) == 0, g);
}

// That of vectors within the row, 32 * VE elements apart, the gradient's 16-byte aligned.
// (A with its near_factor.)
template <typename T, int NV>
__device__ __forceinline__ void store_plain(T* to, const uint4 (&v)[NV], float R, float A, const DistillArgs& a) {
  const float2 c2 = make_float2(a.c, a.c), lo2 = make_float2(a.c_lo, a.c_lo), r2 = make_float2(-R, -R);
#pragma unroll
  for (int i = 0; i < NV; ++i) *(uint4*)(to + i * 32 * Elem<T>::VE) = grad_vec<T>(v[i], c2, lo2, r2, A);
}

// A list warp's work on a row: teacher probabilities, equal tokens, the listed tokens' terms.
template <typename T>
__device__ __forceinline__ void list_part(ListBuf& sh, const DistillArgs& a, long long n, int lane) {
  const double inf = (double)pos_inf(), invT = 1.0 / a.T;
  const T* row = (const T*)a.logits + (long long)n * a.ld;
  double mt = -inf;
  float mx = neg_inf();
  for (int i = lane; i < HASH; i += 32) sh.hash[i] = -1;
#pragma unroll 2
  for (int j = lane; j < a.k; j += 32) {
    const int32_t id = a.idx[n * a.idx_ld + j];
    const double t = teacher_value(a, n, j) * invT;
    const bool in = id >= 0 && id < a.V;
    const float x = in ? Elem<T>::load(row, id) : neg_inf();
    sh.idx[j] = in ? id : -1;
    sh.x[j] = x;
    sh.q[j] = in ? t : -inf;
    if (in) {
      mt = !(t <= mt) ? t : mt;  // NaN is taken over
      mx = fmaxf(mx, x);
    }
  }
  mx = warp_max(mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double y = __shfl_xor_sync(FULL, mt, o);
    mt = mt != mt ? mt : !(y <= mt) ? y : mt;
  }
  // q = exp(t - norm): of the whole vocabulary's sum, or first of the largest
  double norm = a.teacher_lse ? (double)a.teacher_lse[n] : mt != -inf ? mt : 0.0;
  double Q = 0.0, ms = 0.0;
  bool dup = false;
  __syncwarp();
  for (int j = lane; j < a.k; j += 32) {
    const int32_t id = sh.idx[j];
    double q = 0.0, e = 0.0;
    bool mine = false;
    if (id >= 0) {
      q = exp(sh.q[j] - norm);
      e = exact_term(sh.x[j], mx, a);
      uint32_t h = ((uint32_t)id * 2654435761u) >> 23;
      for (;;) {
        const int32_t had = atomicCAS(&sh.hash[h], -1, id);
        mine = had == -1;
        if (had == -1 || had == id) break;
        h = (h + 1) & (HASH - 1);
      }
      dup = dup || !mine;
      ms += mine ? e : 0.0;
    }
    sh.q[j] = q;
    sh.e[j] = e;
    sh.first[j] = mine;
    Q += q;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Q += __shfl_xor_sync(FULL, Q, o);
    ms += __shfl_xor_sync(FULL, ms, o);
  }
  double per = 1.0;
  if (!a.teacher_lse && Q != 0.0) {
    per = 1.0 / Q;
    norm += log(Q);
    Q *= per;
  }
  dup = __any_sync(FULL, dup);
  if (!a.teacher_lse)
    for (int j = lane; j < a.k; j += 32) sh.q[j] *= per;
  __syncwarp();
  for (int j = lane; j < a.k; j += 32) {
    double s = sh.q[j];
    if (dup && sh.idx[j] >= 0) {
      // a token listed more than once: its first entry stands for all
      s = 0.0;
      bool first = true;
      for (int o = 0; o < a.k; ++o)
        if (sh.idx[o] == sh.idx[j]) {
          s += sh.q[o];
          first = first && o >= j;
        }
      sh.first[j] = first;
    }
    sh.qs[j] = s;
  }
  if (lane == 0) {
    const double rest = 1.0 - Q;
    sh.Q = Q;
    sh.norm = norm;
    sh.rest = a.teacher_lse ? (rest < 0.0 ? 0.0 : rest) : 0.0;
    sh.member = Partial{mx, ms};
  }
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(ROW_THREADS, 2) distill_row_kernel(const __grid_constant__ DistillArgs a) {
  extern __shared__ uint4 ring[];
  __shared__ RowShared sh;
  constexpr int VE = Elem<T>::VE, SEG = 32 * VE;
  constexpr int WORKERS = (ROW_WARPS + 1) * 32;  // the streaming warps and one other
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const uint32_t csize = cluster_size(), crank = cluster_rank();
  const bool tail = a.teacher_lse != nullptr;
  if (csize > 1) {
    if (tid < 2) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(&sh.arrived[tid])),
                   "r"(csize)
                   : "memory");
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    cluster_arrive();
    cluster_wait();
  }
  RowWalk rows(blockIdx.x / csize, gridDim.x / csize);
  int p = 0;

  if (wid < ROW_WARPS) {
    const int part = (int)crank * ROW_WARPS + wid;
    uint4* slots = ring + wid * a.ring_segs * 32 + lane;
    const uint32_t slots_at = (uint32_t)__cvta_generic_to_shared(slots);
    constexpr int slot_vecs = BATCH * 32;
    const int batches = a.batches;
    auto zeros = [&](int n) {
      if (GRAD) {
        const Part<T> t(a, n, part, lane);
        T* grow = (T*)a.grad + (long long)n * a.grad_ld;
        for (int i = 0; i < t.segs; ++i)
          store_vec<T>(grow, t.lo + i * SEG, a.V, row_head<T>(grow) == row_head<T>(t.row), make_uint4(0, 0, 0, 0));
      }
    };
    int row = rows.next(a, zeros);
    // batches of a row that pass through the ring: once, or once more for the gradient
    const int passes = GRAD && !a.keep ? 2 * batches : batches;
    Part<T> here(a, max(row, 0), part, lane);
    if (row >= 0)
      for (int i = 0; i < a.slots; ++i) here.copy(a, i >= batches ? i - batches : i, slots_at + i * slot_vecs * 16);
    int slot = 0;
    while (row >= 0) {
      const int after = rows.next(a, zeros);
      const Part<T> then(a, max(after, 0), part, lane);
      // the batch that takes a freed slot: `slots` ahead in this row, or of the next one
      auto refill = [&](int pass, int to) {
        int q = pass + a.slots;
        const uint32_t at = slots_at + to * slot_vecs * 16;
        if (q < passes) {
          here.copy(a, q >= batches ? q - batches : q, at);
        } else if (after >= 0) {
          q -= passes;
          then.copy(a, q >= batches ? q - batches : q, at);
        } else {
          copies_commit();
        }
      };
      bar_sync(BAR_FULL + p, WORKERS);
      Partial acc{neg_inf(), 0.0};
      auto add_terms = [&](const auto& v, float most) {
        const float m = fmaxf(acc.m, warp_max(most));
        acc.s = acc.s * ref_scale(acc.m, m, a.c) + (double)sum_terms<T>(v, m, a);
        acc.m = m;
      };
      for (int b = 0; b < batches; ++b) {
        uint4* at = slots + slot * slot_vecs;
        const int n = here.count(b);
        copies_wait(a.keep ? batches - 1 - b : a.slots - 1);
        here.settle(a, b, at);
        if (tail) here.leave_out(a, b, sh.list[p].idx, at, lane);
        if (n == BATCH) {
          uint4 v[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) v[i] = at[i * 32];
          float m = Elem<T>::vec_max(v[0]);
#pragma unroll
          for (int i = 1; i < BATCH; ++i) m = fmaxf(m, Elem<T>::vec_max(v[i]));
          add_terms(v, m);
        } else {
#pragma unroll 1
          for (int i = 0; i < n; ++i) {
            const uint4 v[1] = {at[i * 32]};
            add_terms(v, Elem<T>::vec_max(v[0]));
          }
        }
        if (!a.keep) refill(b, slot);
        if (++slot == a.slots) slot = 0;
      }
      acc.s = warp_reduce_add(acc.s);  // every lane has the same reference
      if (lane == 0) sh.warp[p][wid] = acc;
      bar_arrive(BAR_SUMS + p, WORKERS);
      if (GRAD) {
        bar_sync(BAR_ROW, WORKERS);
        const float m = sh.m_s, f = sh.A, near = near_factor<T>(f, m, a), R = reference(m, a.c);
        T* grow = (T*)a.grad + (long long)row * a.grad_ld;
        const bool plain =
            here.inside && row_head<T>(grow) == row_head<T>(here.row) && !(m > neg_inf() && is_far(m, a.c));
        for (int b = 0; b < batches; ++b) {
          uint4* at = slots + slot * slot_vecs;
          const int n = here.count(b), lo = here.lo + b * BATCH * SEG;
          if (!a.keep) {
            copies_wait(a.slots - 1);
            here.settle(a, b, at);
          }
          if (plain && n == BATCH) {
            uint4 v[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) v[i] = at[i * 32];
            store_plain<T>(grow + lo, v, R, near, a);
          } else {
#pragma unroll 1
            for (int i = 0; i < n; ++i) store_any<T>(grow, at[i * 32], lo + i * SEG, a.V, m, f, a);
          }
          refill(a.keep ? b : batches + b, slot);
          if (++slot == a.slots) slot = 0;
        }
        bar_arrive(BAR_DONE, WORKERS);
      }
      row = after;
      here = then;
      p ^= 1;
    }
  } else if (wid == JOIN_WARP) {
    uint32_t phase = 0;  // bit p: parity of arrived[p]
    auto none_lost = [&](int n) {
      if (crank == 0 && lane == 0) a.loss[n] = 0.0f;
    };
    for (int n = rows.next(a, none_lost); n >= 0; n = rows.next(a, none_lost)) {
      const double w = a.weight ? (double)a.weight[n] : 1.0;
      ListBuf& list = sh.list[p];
      bar_sync(BAR_SUMS + p, WORKERS);
      Partial s{neg_inf(), 0.0};
      if (lane < ROW_WARPS) s = sh.warp[p][lane];
      s = warp_join(s, a.c);
      bool lost = false;
      if (csize > 1) {
        if (lane < csize) send_partial(&sh.cta[p][crank], &sh.arrived[p], lane, s);
        lost = !wait_partials(&sh.arrived[p], (phase >> p) & 1u);
        phase ^= 1u << p;
        s = Partial{neg_inf(), 0.0};
        if (lane < csize) s = sh.cta[p][lane];
        s = warp_join(s, a.c);
      }
      // all tokens: what was streamed, and the listed ones where they were left out
      const double pos = (double)pos_inf();
      const float m_all = tail ? fmaxf(s.m, list.member.m) : s.m;
      const double scale = ref_scale(s.m, m_all, a.c);
      double e_scale = ref_scale(list.member.m, m_all, a.c);
      double S = s.s * scale + (tail ? list.member.s * e_scale : 0.0);
      if (m_all == pos_inf() || lost) S = pos - pos;  // +inf logits have no softmax: NaN
      double q_t = list.rest;
      if (s.s == 0.0 || scale == 0.0) q_t = q_t == q_t ? 0.0 : q_t;  // no unlisted token with a probability (in 64 bits)
      const double total = list.Q + q_t;
      // outside the list: grad = A * 2^(x C - Rs)
      double A = S;
      if (S == S) A = s.s > 0.0 ? a.T * (total * scale / S - (q_t != 0.0 ? q_t / s.s : 0.0)) : 0.0;
      if (GRAD) {
        if (lane == 0) {
          sh.A = (float)(A * w);
          sh.m_s = s.m;
        }
        bar_arrive(BAR_ROW, WORKERS);
      }
      // log sum exp((x - m_all)/T); a row of -inf alone has none
      if (crank == 0) {
        const bool none = !(m_all > neg_inf()) && S == S;
        const bool far = !none && is_far(m_all, a.c);
        const double logS =
            none ? 0.0 : far ? log(S) : ONE_LN2 * (log2(S) - ((double)m_all * a.C - (double)reference(m_all, a.c)));
        const double invT = 1.0 / a.T;
        double l = 0.0;
        for (int j = lane; j < a.k; j += 32) {
          const double q = list.q[j];
          if (list.idx[j] >= 0 && q != 0.0) {
            const double x = (double)list.x[j];
            const double logp = none || x == -pos ? (S == S ? -pos : S) : (x - (double)m_all) * invT - logS;
            l += q * ((teacher_value(a, n, j) * invT - list.norm) - logp);
          }
        }
        l = warp_reduce_add(l);
        // p_t = s.s * scale / S
        if (q_t != 0.0) l += q_t * (log(q_t) - (log(s.s) + log(scale) - log(S)));
        if (S != S) l = S;
        if (lane == 0) {
          a.loss[n] = (float)(w * a.T * a.T * l);
          if (a.stats) {
            double* st = a.stats + (long long)n * STATS;
            st[ST_MS] = (double)s.m;
            st[ST_A] = A;
            st[ST_LOGQ] = list.norm;
            st[ST_TOTAL] = total;
            st[ST_MALL] = (double)m_all;
            st[ST_LOGS] = logS;
          }
        }
      }
      if (GRAD) {
        // the listed places of this CTA's part, behind the rest of it
        e_scale = S == 0.0 ? 0.0 : e_scale / S;  // from e to p
        const long long head = row_head<T>((const T*)a.logits + (long long)n * a.ld);
        const long long from = (long long)crank * ROW_WARPS * a.warp_segs * SEG - head;
        const long long to = from + (long long)ROW_WARPS * a.warp_segs * SEG;
        T* grow = (T*)a.grad + (long long)n * a.grad_ld;
        bar_sync(BAR_DONE, WORKERS);
        for (int j = lane; j < a.k; j += 32) {
          const long long id = list.idx[j];
          if (id >= 0 && list.first[j] && id >= from && id < to)
            Elem<T>::store(grow, id, (float)(w * a.T * (total * (list.e[j] * e_scale) - list.qs[j])));
        }
      }
      bar_arrive(BAR_EMPTY + p, 64);
      p ^= 1;
    }
  } else {
    auto nothing = [](int) {};
    int done = 0;
    for (int n = rows.next(a, nothing); n >= 0; n = rows.next(a, nothing), p ^= 1) {
      if (done++ > 1) bar_sync(BAR_EMPTY + p, 64);
      list_part<T>(sh.list[p], a, n, lane);
      bar_arrive(BAR_FULL + p, WORKERS);
    }
    // the last rows' sign-offs have no other taker
    if (done > 1) bar_sync(BAR_EMPTY + p, 64);
    if (done > 0) bar_sync(BAR_EMPTY + (p ^ 1), 64);
  }
  if (csize > 1) {
    cluster_arrive();
    cluster_wait();
  }
}

// Zeros for units [ua, ub) of a gradient row.
template <typename T>
__device__ __forceinline__ void zero_units(T* grow, int head, long long V, bool vec, long long ua, long long ub) {
  const uint4 z = make_uint4(0, 0, 0, 0);
  for (long long s = ua * UNIT_SLOTS + threadIdx.x; s < ub * UNIT_SLOTS; s += blockDim.x)
    store_vec<T>(grow, s * Elem<T>::VE - head, V, vec, z);
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
  const T* row = (const T*)a.logits + (long long)n * a.ld;
  T* grow = (T*)a.grad + (long long)n * a.grad_ld;
  const int head = row_head<T>(row);
  const bool vec = row_head<T>(grow) == head;
  const float w = a.weight ? a.weight[n] : 1.0f;
  if (w == 0.0f) {
    zero_units<T>(grow, head, a.V, vec, ua, ub);
    return;
  }
  if (tid == 0) count = 0;
  __syncthreads();
  const double* st = a.stats + (long long)n * STATS;
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
  if (u < ub) {
    const long long lo = (u * UNIT_SLOTS + lane) * VE - head, part = lo - lane * VE;
    if (vec && part >= 0 && part + UNIT_SLOTS * VE <= a.V && !(m > neg_inf() && is_far(m, a.c))) {
      store_plain<T>(grow + lo, v, reference(m, a.c), near_factor<T>(A, m, a), a);
    } else {
#pragma unroll
      for (int i = 0; i < UNIT_VECS; ++i)
        if (lo + i * 32 * VE < a.V) store_any<T>(grow, v[i], lo + i * 32 * VE, a.V, m, A, a);
    }
  }
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
