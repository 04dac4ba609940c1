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
// A row's units (pesti_rowscan.cuh: 4 KB, held by one warp in registers) pass
// through three steps, each a device function of one warp:
//   scan_unit    the unit's largest logit and its sum of terms.  With q_t, listed
//                tokens are left out: p_t is summed from the unlisted tokens
//                themselves, since 1 - sum p would lose it when the list holds
//                nearly all the mass;
//   list_row     what a row's list gives by itself: teacher probabilities, listed
//                tokens' terms, equal tokens (in the scans' grid, beside them);
//   join_row     joins a row's units and its list: loss, the row's factor A and
//                the gradients of its listed tokens;
//   grad_unit    the gradient of a unit.
// Loss: a kernel of scans and lists, then one of joins.  The gradient: one kernel
// more, so large calls read the logits from HBM twice.
//
// Sums: 64 terms of a lane and unit in f32, lanes in 64 bits, a unit's sum
// rounded to f32 once, units in 64 bits, all in a fixed order.  Everything of the
// list (k <= 256 entries) is in 64 bits: the loss is a difference of nearly equal
// logarithms.
#pragma once
#include "pesti_common.cuh"
#include "pesti_rowscan.cuh"

namespace pesti_rows {

constexpr int MAX_TOP = 256;
constexpr int HASH = 512;
constexpr int STATS = 8;       // numbers of a row, and then its list's gradients
constexpr int UNIT_WARPS = 4;  // warps of a block, a unit each
// |m*c| from which on only a row's largest logit counts (pesti_rowscan.cuh).  Below it m*c_lo is at most 2^-23 * 2^29 =
// 64 and R's rounding 16, so that terms stay within 2^+-80; with 2^30 they would leave f32.  The next smaller f32 lies
// 32 powers of two below.
constexpr float FAR_SPLIT = 536870912.0f;
constexpr double ONE_LN2 = 0.69314718055994530942;

__host__ __device__ __forceinline__ long long stats_of(int k) { return STATS + k; }

// What the gradient needs of a row.
enum { ST_MS = 0, ST_A = 1 };

// A unit's largest logit (never NaN) and its sum of terms relative to it.
struct __align__(8) Partial {
  float m, s;
};

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
  float c, c_lo;  // C = c + c_lo, 0 < c_lo <= 2^-23 C
  float* loss;
  double* stats;  // [N][stats_of(k)], null when no gradient follows
  void* grad;
  long long grad_ld;
  long long N, units;
  const float* up;  // none: 1
  long long up_stride;
  Partial* parts;  // [N][units]
  double* lists;   // [N][lists_of(k)]
};

// What list_row leaves of a row: numbers, then e = 2^(x C - R) for the largest listed logit's R and the sum of q over
// equal tokens of every entry (0 where there is none).
enum { LI_Q = 0, LI_LOSS = 1, LI_TERMS = 2, LI_MOST = 3, LI_ENTRIES = 4 };
__host__ __device__ __forceinline__ long long lists_of(int k) { return LI_ENTRIES + 2 * k; }

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
  if (is_far(m, a.c, FAR_SPLIT)) return x == m ? 1.0 : 0.0;
  return exp2((double)x * a.C - (double)ceilf(m * a.c));
}

// The reference R of a row's or unit's largest logit m (0 where it is not used).
__device__ __forceinline__ float reference(float m, float c) {
  return m > neg_inf() && !is_far(m, c, FAR_SPLIT) ? ceilf(m * c) : 0.0f;
}

// A term where m is far: 1 at m itself.
__device__ __forceinline__ float far_term(float x, float m) { return x == m ? 1.0f : x != x ? x : 0.0f; }

// Sum of a lane's terms.
template <typename T, int NV>
__device__ __forceinline__ float sum_terms(const uint4 (&v)[NV], float m, const DistillArgs& a) {
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
  if (m > neg_inf() && is_far(m, a.c, FAR_SPLIT)) {
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
// |(x - m) c_lo| <= 2^-23 |(x - m) C|, is far below their rounding.
template <typename T>
__device__ __forceinline__ float near_factor(float A, float m, const DistillArgs& a) {
  return sizeof(T) == 2 && m > neg_inf() && !is_far(m, a.c, FAR_SPLIT) ? A * ex2(m * a.c_lo) : A;
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
  if (m > neg_inf() && is_far(m, a.c, FAR_SPLIT)) {
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

// Sets the listed elements of a unit (`first` is its first element) to -inf in the lanes' registers.  (By a mask of the
// lane's 64 elements: an index into v would put it into local memory.)
template <typename T>
__device__ __forceinline__ void leave_out(uint4 (&v)[UNIT_VECS], const DistillArgs& a, long long n, long long first,
                                          int lane) {
  constexpr int VE = Elem<T>::VE;
  const int32_t* idx = a.idx + n * a.idx_ld;
  unsigned long long mine = 0ull;
  for (int j0 = 0; j0 < a.k; j0 += 32) {
    const int id = j0 + lane < a.k ? idx[j0 + lane] : -1;
    const long long o = (long long)id - first;
    uint32_t in = __ballot_sync(FULL, id >= 0 && id < a.V && o >= 0 && o < UNIT_SLOTS * VE);
    while (in) {
      const int e = __shfl_sync(FULL, (int)o, __ffs(in) - 1);
      in &= in - 1;
      if (lane == ((e / VE) & 31)) mine |= 1ull << (e / (32 * VE) * VE + e % VE);
    }
  }
  if (!__any_sync(FULL, mine != 0ull)) return;
#pragma unroll
  for (int i = 0; i < UNIT_VECS; ++i) {
    const uint32_t m = (uint32_t)(mine >> (i * VE)) & ((1u << VE) - 1u);
    if (__any_sync(FULL, m)) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        uint4 w = v[i];
        Elem<T>::put(w, e, Elem<T>::NEG_INF);
        if ((m >> e) & 1u) v[i] = w;
      }
    }
  }
}

// A unit's part of its row's sum.
template <typename T>
__device__ __forceinline__ Partial scan_unit(const DistillArgs& a, long long n, long long u, int lane) {
  const T* row = (const T*)a.logits + n * a.ld;
  const int head = row_head<T>(row);
  uint4 v[UNIT_VECS];
  load_unit<T, true>(v, row, head, a.V, u, lane);
  if (a.teacher_lse) leave_out<T>(v, a, n, u * UNIT_SLOTS * Elem<T>::VE - head, lane);
  float m = Elem<T>::vec_max(v[0]);
#pragma unroll
  for (int i = 1; i < UNIT_VECS; ++i) m = fmaxf(m, Elem<T>::vec_max(v[i]));
  Partial p;
  p.m = fmaxf(warp_max(m), neg_inf());  // NaN alone: -inf, with a sum of NaN
  p.s = (float)warp_reduce_add((double)sum_terms<T>(v, p.m, a));
  return p;
}

// A row's list, by one warp.  `hash` (HASH words of shared memory) finds equal tokens.
template <typename T>
__device__ __forceinline__ void list_row(const DistillArgs& a, long long n, int32_t* hash, int lane) {
  const double inf = (double)pos_inf(), invT = 1.0 / a.T;
  const bool tail = a.teacher_lse != nullptr;
  const T* row = (const T*)a.logits + n * a.ld;
  const int32_t* idx = a.idx + n * a.idx_ld;
  double* out = a.lists + n * lists_of(a.k);
  auto listed = [&](int j) {  // the token of entry j, -1 if there is none
    const int32_t id = j < a.k ? idx[j] : -1;
    return id >= 0 && id < a.V ? id : -1;
  };
  for (int i = lane; i < HASH; i += 32) hash[i] = -1;
  __syncwarp();
  // the largest teacher value and listed logit
  double mt = -inf;
  float mx = neg_inf();
#pragma unroll 4
  for (int j = lane; j < a.k; j += 32) {
    const int32_t id = listed(j);
    const double t = teacher_value(a, n, j) * invT;
    if (id >= 0) {
      mt = !(t <= mt) ? t : mt;  // NaN is taken over
      mx = fmaxf(mx, Elem<T>::load(row, id));
    }
  }
  mx = warp_max(mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double y = __shfl_xor_sync(FULL, mt, o);
    mt = mt != mt ? mt : !(y <= mt) ? y : mt;
  }
  // q = exp(t - ref): of the whole vocabulary's sum, or first of the largest; listed tokens' terms, each token once
  const double ref = tail ? (double)a.teacher_lse[n] : mt != -inf ? mt : 0.0;
  double Q = 0.0, terms = 0.0, l = 0.0;
  bool twice = false;  // a token is listed more than once
  for (int j0 = 0; j0 < a.k; j0 += 32) {
    const int j = j0 + lane;
    const int32_t id = listed(j);
    bool first = false;  // this entry stands for its token
    if (id >= 0) {
      uint32_t h = ((uint32_t)id * 2654435761u) >> 23;
      for (;;) {
        const int32_t had = atomicCAS(hash + h, -1, id);
        first = had == -1;
        if (had == -1 || had == id) break;
        h = (h + 1) & (HASH - 1);
      }
    }
    twice = twice || (id >= 0 && !first);
    if (j < a.k) {
      double q = 0.0, e = 0.0;
      if (id >= 0) {
        const float x = Elem<T>::load(row, id);
        const double logq = teacher_value(a, n, j) * invT - ref;
        q = exp(logq);
        e = exact_term(x, mx, a);
        if (q != 0.0) l += q * (logq - (x == neg_inf() ? -inf : ((double)x - (double)mx) * invT));
        Q += q;
        terms += first ? e : 0.0;
      }
      out[LI_ENTRIES + j] = e;
      out[LI_ENTRIES + a.k + j] = q;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Q += __shfl_xor_sync(FULL, Q, o);
    terms += __shfl_xor_sync(FULL, terms, o);
    l += __shfl_xor_sync(FULL, l, o);
  }
  double per = 1.0;
  if (!tail && Q != 0.0) {
    // q, and sum q log q, for the sum Q of the exponentials: log q = t - ref - log Q
    per = 1.0 / Q;
    l = l * per - log(Q);
    Q = Q == Q ? 1.0 : Q;
  }
  twice = __any_sync(FULL, twice);
  if (twice || !tail) {
    __syncwarp();
    for (int j0 = 0; j0 < a.k; j0 += 32) {
      const int j = j0 + lane;
      const int32_t id = listed(j);
      if (j < a.k) {
        double s = out[LI_ENTRIES + a.k + j];
        if (twice && id >= 0) {
          // every entry of a token gets the token's sum
          s = 0.0;
          for (int o = 0; o < a.k; ++o)
            if (idx[o] == id) s += exp(teacher_value(a, n, o) * invT - ref);
        }
        out[LI_ENTRIES + a.k + j] = s * per;
      }
    }
  }
  if (lane == 0) {
    out[LI_Q] = Q;
    out[LI_LOSS] = l;
    out[LI_TERMS] = terms;
    out[LI_MOST] = (double)mx;
  }
}

// A row's loss, and its numbers for the gradient, by one warp.
template <typename T>
__device__ __forceinline__ void join_row(const DistillArgs& a, long long n, int lane) {
  const double inf = (double)pos_inf(), w = a.weight ? (double)a.weight[n] : 1.0;
  const bool tail = a.teacher_lse != nullptr;
  const double* list = a.lists + n * lists_of(a.k);
  const Partial* parts = a.parts + n * a.units;
  const double Q = list[LI_Q], l0 = list[LI_LOSS], terms = list[LI_TERMS];
  const float mx = (float)list[LI_MOST];
  // what was scanned
  float m_s = neg_inf();
  double s = 0.0;
#pragma unroll 4
  for (long long u = lane; u < a.units; u += 32) m_s = fmaxf(m_s, parts[u].m);
  m_s = warp_max(m_s);
#pragma unroll 4
  for (long long u = lane; u < a.units; u += 32) {
    const Partial p = parts[u];
    s += (double)p.s * ref_scale(p.m, m_s, a.c, FAR_SPLIT);
  }
  s = warp_reduce_add(s);
  // all tokens: what was scanned, and the listed ones where they were left out
  const float m_all = tail ? fmaxf(m_s, mx) : m_s;
  const double scale = ref_scale(m_s, m_all, a.c, FAR_SPLIT), e_scale = ref_scale(mx, m_all, a.c, FAR_SPLIT);
  double S = s * scale + (tail ? terms * e_scale : 0.0);
  if (m_all == pos_inf()) S = inf - inf;  // +inf logits have no softmax: NaN
  const double rest = 1.0 - Q;
  double q_t = tail ? (rest < 0.0 ? 0.0 : rest) : 0.0;
  if (s == 0.0 || scale == 0.0) q_t = q_t == q_t ? 0.0 : q_t;  // no unlisted token with a probability (in 64 bits)
  const double total = Q + q_t;
  if (a.stats) {
    double* st = a.stats + n * stats_of(a.k);
    // outside the list: grad = A * 2^(x C - Rs)
    double A = S;
    if (S == S) A = s > 0.0 ? a.T * (total * scale / S - (q_t != 0.0 ? q_t / s : 0.0)) : 0.0;
    if (lane == 0) {
      st[ST_MS] = (double)m_s;
      st[ST_A] = A;
    }
    // p of a listed token is e * to_p; a row of -inf alone has none
    const double to_p = S == 0.0 ? 0.0 : e_scale / S;
    for (int j = lane; j < a.k; j += 32)
      st[STATS + j] = a.T * (total * (list[LI_ENTRIES + j] * to_p) - list[LI_ENTRIES + a.k + j]);
  }
  if (lane == 0) {
    // sum q (log q - (x - mx)/T) + Q (log sum exp of (x - mx)/T) + q_t (log q_t - log p_t), p_t = s * scale / S
    double l = l0;
    if (m_all > neg_inf() && Q != 0.0) {
      const double lse =
          is_far(m_all, a.c, FAR_SPLIT)
              ? log(S)
              : ONE_LN2 * (log2(S) - ((double)m_all * a.C - (double)reference(m_all, a.c)));
      l += Q * (((double)m_all - (double)mx) / a.T + lse);
    }
    if (q_t != 0.0) l += q_t * (log(q_t) - log(s * scale / S));
    if (S != S) l = S;
    a.loss[n] = (float)(w * a.T * a.T * l);
  }
}

// Stores a unit's gradient vectors whose elements start d (1 to VE - 1) places before a 16-byte boundary of the
// gradient: each lane writes the vector that its own and the next lane's make up, the unit's ragged ends go one by one.
// (Loss and gradient of 461 rows of 256000 bf16 whose logits are padded by one: 134 us, 333 us with single elements.)
template <typename T>
__device__ __forceinline__ void store_shifted(T* to, const uint4 (&g)[UNIT_VECS], int d, int lane) {
  constexpr int VE = Elem<T>::VE;
  const int words = d * (int)sizeof(T) / 4, bits = d * (int)sizeof(T) % 4 * 8;
#pragma unroll
  for (int i = 0; i < UNIT_VECS; ++i) {
    // lane 31's neighbour is lane 0 of the next vectors
    const uint4 out = lane == 0 && i + 1 < UNIT_VECS ? g[i + 1 < UNIT_VECS ? i + 1 : i] : g[i];
    const int next = (lane + 1) & 31;
    const uint32_t w[8] = {g[i].x,
                           g[i].y,
                           g[i].z,
                           g[i].w,
                           __shfl_sync(FULL, out.x, next),
                           __shfl_sync(FULL, out.y, next),
                           __shfl_sync(FULL, out.z, next),
                           __shfl_sync(FULL, out.w, next)};
    uint32_t r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t lo = w[k], hi = w[k + 1];
      if (words == 1) lo = w[k + 1], hi = w[k + 2 < 8 ? k + 2 : 7];
      if (words == 2) lo = w[k + 2], hi = w[k + 3 < 8 ? k + 3 : 7];
      if (words == 3) lo = w[k + 3], hi = w[k + 4 < 8 ? k + 4 : 7];
      r[k] = __funnelshift_r(lo, hi, bits);
    }
    if (i + 1 < UNIT_VECS || lane < 31) *(uint4*)(to + i * 32 * VE + d) = make_uint4(r[0], r[1], r[2], r[3]);
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    if (lane == 0 && e < d) Elem<T>::store(to, e, Elem<T>::at(g[0], e));
    if (lane == 31 && e >= d) Elem<T>::store(to + (UNIT_VECS - 1) * 32 * VE, e, Elem<T>::at(g[UNIT_VECS - 1], e));
  }
}

// The gradient of a unit, in place too: everything is read before anything is written.
template <typename T>
__device__ __forceinline__ void grad_unit(const DistillArgs& a, long long n, long long u, double scale, int lane) {
  constexpr int VE = Elem<T>::VE;
  const T* row = (const T*)a.logits + n * a.ld;
  T* grow = (T*)a.grad + n * a.grad_ld;
  const int head = row_head<T>(row);
  uint4 v[UNIT_VECS];
  load_unit<T, false>(v, row, head, a.V, u, lane);
  const double* st = a.stats + n * stats_of(a.k);
  const float m = (float)__ldcg(st + ST_MS), A = (float)(__ldcg(st + ST_A) * scale);
  const long long first = u * UNIT_SLOTS * VE - head, lo = first + lane * VE;
  constexpr int span = UNIT_SLOTS * VE;
  __syncwarp();
  const bool inner = first >= 0 && first + span <= a.V && !(m > neg_inf() && is_far(m, a.c, FAR_SPLIT));
  const int past = row_head<T>(grow + lo);  // the vectors' place behind a 16-byte boundary of the gradient
  if (inner) {
    const float R = reference(m, a.c), f = near_factor<T>(A, m, a);
    if (past == 0) {
      store_plain<T>(grow + lo, v, R, f, a);
    } else {
      const float2 c2 = make_float2(a.c, a.c), lo2 = make_float2(a.c_lo, a.c_lo), r2 = make_float2(-R, -R);
#pragma unroll
      for (int i = 0; i < UNIT_VECS; ++i) v[i] = grad_vec<T>(v[i], c2, lo2, r2, f);
      store_shifted<T>(grow + lo, v, VE - past, lane);
    }
  } else {
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i)
      if (lo + i * 32 * VE < a.V) store_any<T>(grow, v[i], lo + i * 32 * VE, a.V, m, A, a);
  }
  // the unit's listed tokens, over what was just written
  __syncwarp();
  const int32_t* idx = a.idx + n * a.idx_ld;
  for (int j = lane; j < a.k; j += 32) {
    const long long id = idx[j];
    if (id >= first && id < first + span && id >= 0 && id < a.V)
      Elem<T>::store(grow, id, (float)(__ldcg(st + STATS + j) * scale));
  }
}

// Zeros for a unit of a row that takes no part.
template <typename T>
__device__ __forceinline__ void zero_unit(const DistillArgs& a, long long n, long long u, int lane) {
  T* grow = (T*)a.grad + n * a.grad_ld;
  const int head = row_head<T>((const T*)a.logits + n * a.ld);
  const bool vec = row_head<T>(grow) == head;
  for (int i = 0; i < UNIT_VECS; ++i)
    store_vec<T>(grow, ((u * UNIT_VECS + i) * 32 + lane) * Elem<T>::VE - head, a.V, vec, make_uint4(0, 0, 0, 0));
}

__device__ __forceinline__ bool takes_part(const DistillArgs& a, long long n) {
  return a.weight == nullptr || a.weight[n] != 0.0f;
}

// The first blocks work on the lists, a warp each; the others on the units.
// (40 warps an SM: 2048 rows of 152064 bf16 take 109 us, 5.7 TB/s; 114 us with the 36 of 54 registers a thread, 124 us
// with blocks of 8 warps.)
template <typename T>
__global__ void __launch_bounds__(UNIT_WARPS * 32, 10) distill_scan_kernel(const __grid_constant__ DistillArgs a,
                                                                       long long list_blocks,
                                                                       long long blocks_per_row) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int32_t hash[UNIT_WARPS][HASH];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  if (blockIdx.x < list_blocks) {
    const long long n = (long long)blockIdx.x * UNIT_WARPS + wid;
    if (n < a.N && takes_part(a, n)) list_row<T>(a, n, hash[wid], lane);
    return;
  }
  const long long block = blockIdx.x - list_blocks, n = block / blocks_per_row;
  const long long u = (block - n * blocks_per_row) * UNIT_WARPS + wid;
  if (u >= a.units || !takes_part(a, n)) return;
  const Partial p = scan_unit<T>(a, n, u, lane);
  if (lane == 0) a.parts[n * a.units + u] = p;
}

constexpr int JOIN_WARPS = 2;  // warps of a block, a row each

// Bound by latency (a row's units, then 64-bit logarithms): 8.4 us for 2048 rows of 152064 bf16, 7 us for 1024 of 128256.
template <typename T>
__global__ void __launch_bounds__(JOIN_WARPS * 32) distill_join_kernel(const __grid_constant__ DistillArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long n = (long long)blockIdx.x * JOIN_WARPS + (threadIdx.x >> 5);
  if (n >= a.N) return;
  if (takes_part(a, n))
    join_row<T>(a, n, threadIdx.x & 31);
  else if ((threadIdx.x & 31) == 0)
    a.loss[n] = 0.0f;
}

// (32 warps an SM: 2048 rows of 152064 bf16 take 168 us, 7.4 TB/s of which some comes from L2.)
template <typename T>
__global__ void __launch_bounds__(UNIT_WARPS * 32, 8) distill_backward_kernel(const __grid_constant__ DistillArgs a,
                                                                           long long blocks_per_row) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long n = blockIdx.x / blocks_per_row;
  const long long u = (blockIdx.x - n * blocks_per_row) * UNIT_WARPS + (threadIdx.x >> 5);
  if (u >= a.units) return;
  const int lane = threadIdx.x & 31;
  if (!takes_part(a, n)) {
    zero_unit<T>(a, n, u, lane);
    return;
  }
  const double w = a.weight ? (double)a.weight[n] : 1.0;
  grad_unit<T>(a, n, u, w * (a.up ? (double)a.up[n * a.up_stride] : 1.0), lane);
}

}  // namespace pesti_rows
