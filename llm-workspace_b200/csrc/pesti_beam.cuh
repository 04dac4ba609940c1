// Beam search on the device: selection over beams and vocabulary, the loop
// control of the beams, and the reordering of per-beam states.
//
// Selection, for the W beams of a group with cumulative scores cum[w]:
//   logp(w, v)  = (x[w,v] - m_w) - log sum_v exp(x[w,v] - m_w)
//   score(w, v) = cum[w] + logp(w, v)
// and the K best (w, v).  Within a beam the order is that of the logits, so
// the K largest logits of each row (equal ones: lower token first) are all
// that the merge needs, and their order needs no arithmetic.  Only the merge
// across beams compares sums, which it does in 64 bits.
//
//  beam_scan_kernel   the one pass over the logits.  A warp holds a unit
//                     (pesti_rowscan.cuh) in registers and writes the unit's
//                     maximum m and S = sum 2^(x*c - R), c = f32(log2 e),
//                     R = ceil(m*c), and its 8 segment maxima.
//  beam_pick_kernel   one block per row: the K segments with the largest
//                     maxima hold the K largest logits; they are read again
//                     and sorted.  The block that finishes a group last
//                     merges its W lists.
//
// Accuracy of a row's log sum as the scan gives it, relative to the sum:
//   2^x by the hardware 2^-22.5; the rounding of x*c - R (one fused
//   operation): half an ulp of t = x*c - R, ln 2 * 2^-24 * E[|t|], and
//   E[|t|] <= 12 since the entropy of 2048 terms is at most 11 bits and R
//   less than 1 above the largest; c's own
//   rounding 1.34e-8 * E[m - x] (<= ln V <= 22); 23 additions in f32, 2^-24
//   each.  Together below 2.4e-6.  Units are joined in 64 bits.  Two
//   candidates of different beams whose scores differ by less than twice
//   LSE_EPS are therefore not ordered by these sums: the merge adds up their
//   rows again in 64 bits, in index order, and ranks once more.  That is one
//   call in some thousands for random logits.
#pragma once
#include "pesti_common.cuh"
#include "pesti_rowscan.cuh"

namespace pesti_rows {

constexpr int MAX_W = 64;          // beams of a group
constexpr int MAX_K = 128;         // candidates of a group
constexpr int SCAN_WARPS = 8;
constexpr int PICK_THREADS = 256;
constexpr int MAX_SEG_KEYS = 4096; // segment maxima a block holds (wider rows: maxima of runs of segments)
constexpr int MAX_SEL = MAX_K + MAX_K / 2 + 8;
constexpr int LIST_CAP = 3072;     // candidates a block holds
constexpr int RANK_CAP = 256;      // candidates it ranks by counting
constexpr double LSE_EPS = 3e-6;
constexpr float LOG2E_F = 1.44269504088896340736f;
constexpr double LN2 = 0.69314718055994530942;

// Order of f32 values as unsigned integers; -0 counts as +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;  // order_key(-inf); NaN counts as -inf

struct RowTop {
  double ref;   // logp(x) = (x - ref) - logs, or -logs for x = +inf when ref is +inf
  double logs;
  int n;        // entries of the row's list
  int pad;
};

struct BeamWs {
  float2* unit;      // [rows][units] maximum and sum
  uint32_t* seg;     // [rows][units*8] order keys of the segment maxima
  RowTop* top;       // [rows]
  float* x;          // [rows][K]
  int32_t* idx;      // [rows][K]
  uint32_t* arrived; // [G]
};

__device__ __forceinline__ bool beam_running(const float* cum, long long row) {
  return cum == nullptr || cum[row] > neg_inf();
}

template <typename T>
__global__ void __launch_bounds__(SCAN_WARPS * 32) beam_scan_kernel(const T* __restrict__ logits, long long ld,
                                                                    long long V, int W, long long units,
                                                                    long long blocks_per_row, const float* cum,
                                                                    const uint8_t* done, int every_row, BeamWs ws) {
  const long long row = blockIdx.x / blocks_per_row;
  const long long ub = blockIdx.x - row * blocks_per_row;
  const long long g = row / W;
  if (ub == 0 && row == g * W && threadIdx.x == 0) ws.arrived[g] = 0u;
  // rows that take no part are not read
  if (done && done[g]) return;
  if (!every_row && !beam_running(cum, row)) return;
  const int lane = threadIdx.x & 31;
  const long long u = ub * SCAN_WARPS + (threadIdx.x >> 5);
  if (u >= units) return;
  const T* p = logits + row * ld;
  uint4 v[UNIT_VECS];
  load_unit<T, true>(v, p, row_head<T>(p), V, u, lane);
  float m = neg_inf();
  float mine = neg_inf();
#pragma unroll
  for (int i = 0; i < UNIT_VECS; ++i) {
    const float s = warp_max(Elem<T>::vec_max(v[i]));
    m = fmaxf(m, s);  // NaN (a segment of NaN alone) is left out
    if (lane == i) mine = s;
  }
  const bool far = m > neg_inf() && is_far(m, LOG2E_F);
  const float R = m > neg_inf() ? ceilf(m * LOG2E_F) : 0.0f;
  float S;
  {
    const float2 c2 = make_float2(LOG2E_F, LOG2E_F), r2 = make_float2(-R, -R);
    float2 a0 = make_float2(0.f, 0.f), a1 = a0;
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i) {
#pragma unroll
      for (int q = 0; q < Elem<T>::PAIRS; ++q) {
        float2 t = fma2(Elem<T>::pair(v[i], q), c2, r2);
        t.x = ex2(t.x);
        t.y = ex2(t.y);
        if (q & 1)
          a1 = add2(a1, t);
        else
          a0 = add2(a0, t);
      }
    }
    S = warp_reduce_add((a0.x + a0.y) + (a1.x + a1.y));
  }
  if (far || S != S) {
    // the number of maxima, or a sum that leaves NaN out
    S = 0.f;
#pragma unroll 1
    for (int i = 0; i < UNIT_VECS; ++i) {
      const uint4 w = i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : i == 3 ? v[3] : i == 4 ? v[4] : i == 5 ? v[5] : i == 6 ? v[6] : v[7];
      for (int q = 0; q < Elem<T>::PAIRS; ++q) {
        const float2 x = Elem<T>::pair(w, q);
        if (far) {
          S += (x.x == m ? 1.f : 0.f) + (x.y == m ? 1.f : 0.f);
        } else {
          if (x.x == x.x) S += ex2(fmaf(x.x, LOG2E_F, -R));
          if (x.y == x.y) S += ex2(fmaf(x.y, LOG2E_F, -R));
        }
      }
    }
    S = warp_reduce_add(S);
  }
  if (lane < UNIT_VECS) {
    const bool none = !(mine > neg_inf());
    ws.seg[(row * units + u) * UNIT_VECS + lane] = none ? KEY_NEG_INF : order_key(mine);
  }
  if (lane == 0) ws.unit[row * units + u] = make_float2(m, S);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Sum over the block of small counts; `buf` alternates between two rows of 8.
__device__ __forceinline__ int block_count(int c, int (*buf)[PICK_THREADS / 32], int& turn) {
  const int s = __reduce_add_sync(FULL, c);
  if ((threadIdx.x & 31) == 0) buf[turn][threadIdx.x >> 5] = s;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int i = 0; i < PICK_THREADS / 32; ++i) t += buf[turn][i];
  turn ^= 1;
  return t;
}

struct PickShared {
  union {
    struct {
      uint32_t keys[MAX_SEG_KEYS];
      unsigned long long list[LIST_CAP];
    } row;
    struct {
      float x[MAX_W * MAX_K];
    } merge;
  };
  unsigned long long sorted_c[RANK_CAP];
  double ref[MAX_W], logs[MAX_W], cum[MAX_W];
  int n[MAX_W];
  int sel[MAX_SEL];
  int count[2][PICK_THREADS / 32];
  int scan[40];
  double red[40];
  int nsel, nlist, over, last, end;
  unsigned long long flagged;
};

// Appends the elements of segment s with key >= t to the list (at most LIST_CAP; `over` if there are more).
template <typename T>
__device__ __forceinline__ void append_vec(PickShared& sh, const uint4& v, long long first, uint32_t t) {
#pragma unroll
  for (int q = 0; q < Elem<T>::PAIRS; ++q) {
    const float2 x = Elem<T>::pair(v, q);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float f = e ? x.y : x.x;
      const uint32_t k = order_key(f);
      if (f == f && k >= t) {
        const int at = atomicAdd(&sh.nlist, 1);
        if (at < LIST_CAP)
          sh.row.list[at] = ((unsigned long long)k << 32) | (uint32_t)~(uint32_t)(first + q * 2 + e);
        else
          sh.over = 1;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 load_seg_vec(const T* p, int head, long long V, long long seg, int lane,
                                              long long& first) {
  first = (seg * 32 + lane) * Elem<T>::VE - head;
  if (first >= 0 && first + Elem<T>::VE <= V) return __ldg((const uint4*)(p - head) + seg * 32 + lane);
  return load_edge<T>(p, first, V);
}

// Cuts the list to its largest entries: at least K and at most `most` (entries are distinct).
__device__ __forceinline__ void prune_list(PickShared& sh, int K, int most, int& turn) {
  __syncthreads();
  const int n = sh.nlist;
  __syncthreads();  // every thread has read it before the next append
  if (n <= most) return;
  unsigned long long lo = 0, hi = ~0ull;
  while (hi - lo > 1) {
    const unsigned long long mid = lo + (hi - lo) / 2;
    int c = 0;
    for (int i = threadIdx.x; i < n; i += PICK_THREADS) c += sh.row.list[i] >= mid;
    c = block_count(c, sh.count, turn);
    if (c >= K) {
      lo = mid;
      if (c <= most) break;
    } else {
      hi = mid;
    }
  }
  // entries kept move to the front; each thread holds its own first
  unsigned long long mine[LIST_CAP / PICK_THREADS];
#pragma unroll
  for (int j = 0; j < LIST_CAP / PICK_THREADS; ++j) {
    const int i = threadIdx.x + j * PICK_THREADS;
    mine[j] = i < n ? sh.row.list[i] : 0ull;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.nlist = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < LIST_CAP / PICK_THREADS; ++j)
    if (mine[j] != 0ull && mine[j] >= lo) sh.row.list[atomicAdd(&sh.nlist, 1)] = mine[j];
  __syncthreads();
}

__device__ __forceinline__ double beam_score(const PickShared& sh, int w, float x) {
  return sh.ref[w] == (double)pos_inf() ? sh.cum[w] - sh.logs[w] : sh.cum[w] + (((double)x - sh.ref[w]) - sh.logs[w]);
}

// Order-preserving image of a double (no NaN).
__device__ __forceinline__ unsigned long long order_key64(double d) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(d + 0.0);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// Ranks the candidates of the group's lists; those with rank < RANK_CAP go to
// sorted_c as list positions w * K + r.
__device__ __forceinline__ int rank_candidates(PickShared& sh, int W, int K) {
  int total = 0;
  for (int w = 0; w < W; ++w) total += sh.n[w];
  for (int j = threadIdx.x; j < W * K; j += PICK_THREADS) {
    const int w = j / K, r = j - w * K;
    if (r >= sh.n[w]) continue;
    const double s = beam_score(sh, w, sh.merge.x[j]);
    int rank = r;
    for (int o = 0; o < W && rank < RANK_CAP; ++o) {
      if (o == w) continue;
      // entries of beam o ahead of s: equal ones count when o is the lower beam
      int lo = 0, hi = sh.n[o];
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const double q = beam_score(sh, o, sh.merge.x[o * K + mid]);
        if (q > s || (q == s && o < w))
          lo = mid + 1;
        else
          hi = mid;
      }
      rank += lo;
    }
    if (rank < RANK_CAP) sh.sorted_c[rank] = (unsigned long long)j;
  }
  __syncthreads();
  return total;
}

template <typename T>
__global__ void __launch_bounds__(PICK_THREADS) beam_pick_kernel(const T* __restrict__ logits, long long ld,
                                                                 long long V, int W, int K, long long units,
                                                                 const float* cum, const uint8_t* done, int every_row,
                                                                 BeamWs ws, float* out_score, int32_t* out_token,
                                                                 int32_t* out_parent, float* out_lse) {
  __shared__ PickShared sh;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const long long row = blockIdx.x;
  const long long g = row / W;
  int turn = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const bool group_done = done && done[g];
  const bool live = !group_done && beam_running(cum, row);
  const T* p = logits + row * ld;
  const int head = row_head<T>(p);
  if (tid == 0) {
    sh.nsel = 0;
    sh.nlist = 0;
    sh.over = 0;
  }
  double ref = 0.0, logs = 0.0;
  int n = 0;
  if (!group_done && (live || every_row)) {
    // the row's sum, joined from its units in a fixed order
    const float2* unit = ws.unit + row * units;
    float m = neg_inf();
    for (long long u = tid; u < units; u += PICK_THREADS) m = fmaxf(m, unit[u].x);
    m = block_reduce_max(m, (float*)sh.scan);
    const bool inf = m == pos_inf(), none = !(m > neg_inf());
    double s = 0.0;
    for (long long u = tid; u < units; u += PICK_THREADS) {
      const float2 a = unit[u];
      if (a.x > neg_inf()) s += (double)a.y * ref_scale(a.x, m, LOG2E_F);
    }
    s = block_reduce_add(s, sh.red);
    if (!none) {
      // sum 2^(x c - R) = 2^(m c - R) sum 2^((x - m) c)
      ref = (double)m;
      logs = is_far(m, LOG2E_F) ? log(s)
                                : LN2 * (log2(s) - ((double)m * (double)LOG2E_F - (double)ceilf(m * LOG2E_F)));
    }
    if (out_lse && tid == 0) out_lse[row] = none ? neg_inf() : inf ? pos_inf() : (float)(ref + logs);

    if (live && !none) {
      // the segments that hold the K largest logits
      const long long nseg = units * UNIT_VECS;
      const int run = (int)((nseg + MAX_SEG_KEYS - 1) / MAX_SEG_KEYS);
      const int nkeys = (int)((nseg + run - 1) / run);
      const uint32_t* seg = ws.seg + row * nseg;
      int valid = 0;
      for (int i = tid; i < nkeys; i += PICK_THREADS) {
        uint32_t k = KEY_NEG_INF;
        const long long end = min(nseg, (long long)(i + 1) * run);
        for (long long j = (long long)i * run; j < end; ++j) k = max(k, seg[j]);
        sh.row.keys[i] = k;
        valid += k > KEY_NEG_INF;
      }
      valid = block_count(valid, sh.count, turn);
      uint32_t t = KEY_NEG_INF + 1;  // every segment with a finite value
      int above = valid;
      if (valid > K) {
        uint32_t lo = t, hi = order_key(m) + 1;
        const int most = K + K / 2 + 8;
        while (hi - lo > 1 && above > most) {
          const uint32_t mid = lo + (hi - lo) / 2;
          int c = 0;
          for (int i = tid; i < nkeys; i += PICK_THREADS) c += sh.row.keys[i] >= mid;
          c = block_count(c, sh.count, turn);
          if (c >= K) {
            lo = mid;
            above = c;
          } else {
            hi = mid;
          }
        }
        t = lo;
        if (above > most) {
          // many segments share the K-th maximum t: those above it, then the first ones at it
          const int per = (nkeys + PICK_THREADS - 1) / PICK_THREADS;
          const int a = tid * per, b = min(nkeys, a + per);
          int more = 0, same = 0;
          for (int i = a; i < b; ++i) {
            more += sh.row.keys[i] > t;
            same += sh.row.keys[i] == t;
          }
          const int over_t = block_count(more, sh.count, turn);
          int total;
          int before = block_excl_scan_add(same, sh.scan, total);
          for (int i = a; i < b; ++i) {
            const uint32_t k = sh.row.keys[i];
            const bool take = k > t || (k == t && before < K - over_t);
            before += k == t;
            if (take) sh.sel[atomicAdd(&sh.nsel, 1)] = i;
          }
          above = 0;
        }
      }
      __syncthreads();
      if (above > 0) {
        for (int i = tid; i < nkeys; i += PICK_THREADS)
          if (sh.row.keys[i] >= t) sh.sel[atomicAdd(&sh.nsel, 1)] = i;
      }
      __syncthreads();
      // their elements from t up: all at once, or in rounds that keep the list short
      const int nsel = sh.nsel;
      const long long todo = (long long)nsel * run;
      for (int i0 = wid; i0 < todo; i0 += 4 * (PICK_THREADS / 32)) {
        uint4 v[4];
        long long first[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const long long i = i0 + j * (PICK_THREADS / 32);
          if (i < todo) {
            const long long sg = (long long)sh.sel[i / run] * run + i % run;
            if (sg < nseg) v[j] = load_seg_vec<T>(p, head, V, sg, lane, first[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const long long i = i0 + j * (PICK_THREADS / 32);
          if (i < todo && (long long)sh.sel[i / run] * run + i % run < nseg) append_vec<T>(sh, v[j], first[j], t);
        }
      }
      __syncthreads();
      if (sh.over) {
        __syncthreads();
        if (tid == 0) sh.nlist = 0;
        __syncthreads();
        for (long long i0 = 0; i0 < todo; i0 += PICK_THREADS / 32) {
          const long long i = i0 + wid;
          if (i < todo) {
            const long long sg = (long long)sh.sel[i / run] * run + i % run;
            if (sg < nseg) {
              long long first;
              const uint4 v = load_seg_vec<T>(p, head, V, sg, lane, first);
              append_vec<T>(sh, v, first, t);  // at most 2048 more behind at most 1024
            }
          }
          prune_list(sh, K, LIST_CAP - (PICK_THREADS / 32) * 32 * Elem<T>::VE, turn);
        }
      }
      prune_list(sh, K, RANK_CAP, turn);
      const int nl = sh.nlist;
      n = min(nl, K);
      if (tid < nl) {
        const unsigned long long c = sh.row.list[tid];
        int rank = 0;
        for (int j = 0; j < nl; ++j) rank += sh.row.list[j] > c;
        if (rank < K) {
          ws.x[row * K + rank] = key_value((uint32_t)(c >> 32));
          ws.idx[row * K + rank] = (int32_t)~(uint32_t)c;
        }
      }
      if (inf) {
        // only the +inf entries have a probability
        const int here = __syncthreads_count(tid < nl && (uint32_t)(sh.row.list[tid] >> 32) == order_key(pos_inf()));
        n = min(n, here);
      }
    }
  } else if (out_lse && tid == 0) {
    out_lse[row] = neg_inf();
  }
  if (tid == 0) {
    RowTop r;
    r.ref = ref;
    r.logs = logs;
    r.n = n;
    r.pad = 0;
    ws.top[row] = r;
  }
  // the block that finishes the group last merges
  __threadfence();
  __syncthreads();
  if (tid == 0) sh.last = atomicAdd(&ws.arrived[g], 1u) == (uint32_t)(W - 1);
  __syncthreads();
  if (!sh.last) return;
  __threadfence();

  const long long row0 = g * W;
  for (int w = tid; w < W; w += PICK_THREADS) {
    const RowTop* r = ws.top + row0 + w;
    sh.ref[w] = __ldcg(&r->ref);
    sh.logs[w] = __ldcg(&r->logs);
    sh.n[w] = __ldcg(&r->n);
    sh.cum[w] = cum ? (double)cum[row0 + w] : 0.0;
  }
  for (int j = tid; j < W * K; j += PICK_THREADS) sh.merge.x[j] = __ldcg(ws.x + row0 * K + j);
  if (tid == 0) {
    sh.flagged = 0ull;
    sh.end = RANK_CAP;
  }
  __syncthreads();
  const int total = rank_candidates(sh, W, K);
  const int have = min(total, RANK_CAP);
  if (W > 1 && total > 1) {
    // pairs of neighbours whose order the sums do not settle, up to the first clear gap behind the K-th place
    const int i = tid;
    bool near = false, apart = false;
    int wa = 0, wb = 0;
    if (i + 1 < have) {
      wa = (int)sh.sorted_c[i] / K;
      wb = (int)sh.sorted_c[i + 1] / K;
      const double a = beam_score(sh, wa, sh.merge.x[sh.sorted_c[i]]);
      const double b = beam_score(sh, wb, sh.merge.x[sh.sorted_c[i + 1]]);
      near = !(a - b > 2.0 * LSE_EPS) && a < (double)pos_inf();
      apart = wa != wb;
      if (!near && i >= K - 1) atomicMin(&sh.end, i);
    }
    __syncthreads();
    if (near && apart && i < sh.end) atomicOr(&sh.flagged, (1ull << wa) | (1ull << wb));
    // a run that leaves the ranked part: every row
    if (tid == 0 && total > RANK_CAP && sh.end == RANK_CAP) sh.flagged = W == 64 ? ~0ull : (1ull << W) - 1ull;
    __syncthreads();
    const unsigned long long flagged = sh.flagged;
    if (flagged) {
      for (int w = 0; w < W; ++w) {
        if (!((flagged >> w) & 1ull) || sh.n[w] == 0 || sh.ref[w] == (double)pos_inf()) continue;
        const T* q = logits + (row0 + w) * ld;
        const double m = sh.ref[w];
        double s = 0.0;
        for (long long v = tid; v < V; v += PICK_THREADS) {
          const float x = Elem<T>::load(q, v);
          if (x == x) s += exp((double)x - m);
        }
        s = block_reduce_add(s, sh.red);
        if (tid == 0) sh.logs[w] = log(s);
        __syncthreads();
      }
      rank_candidates(sh, W, K);
    }
  }
  for (int r = tid; r < K; r += PICK_THREADS) {
    float sc = neg_inf();
    int tk = -1, pa = -1;
    if (r < total) {
      const int j = (int)sh.sorted_c[r];
      pa = j / K;
      sc = (float)beam_score(sh, pa, sh.merge.x[j]);
      tk = __ldcg(ws.idx + row0 * K + j);
    }
    out_score[g * K + r] = sc;
    out_token[g * K + r] = tk;
    out_parent[g * K + r] = pa;
  }
}

// ---------------------------------------------------------------- loop control

struct BeamStatePtrs {
  float* cum;
  int32_t* last;
  int32_t* parent;
  int32_t* tokens;
  int32_t* count;
  uint8_t* done;
  int32_t* fin_tokens;
  int32_t* fin_len;
  float* fin_score;
  int32_t* fin_count;
  long long cap;
};

constexpr int ADV_THREADS = 128;

// One block per group.  The ranks are walked by one thread: which candidates
// end, which go on, and which slots of the pool they take.  The block then
// moves the token histories: a thread owns a column of all beams, so rows
// exchange places without another buffer.
__global__ void __launch_bounds__(ADV_THREADS) beam_advance_kernel(const float* __restrict__ score,
                                                                   const int32_t* __restrict__ token,
                                                                   const int32_t* __restrict__ parent, int W, int K,
                                                                   const uint32_t* __restrict__ stop, long long n_stop,
                                                                   long long max_tokens, long long max_seq_len,
                                                                   double alpha, int early, BeamStatePtrs st) {
  extern __shared__ int32_t tile[];  // [W][ADV_THREADS]
  __shared__ uint8_t is_stop[MAX_K];
  __shared__ float cand_s[MAX_K];
  __shared__ int32_t cand_t[MAX_K], cand_p[MAX_K];
  __shared__ float fin_score[MAX_W], new_cum[MAX_W];
  __shared__ int32_t fin_len[MAX_W], src[MAX_W], new_par[MAX_W], new_tok[MAX_W];
  __shared__ double len_pow[3];
  __shared__ int live_n, fin_n, code;
  const long long g = blockIdx.x;
  const int tid = threadIdx.x;
  const long long limit = min(max_tokens, max_seq_len);
  if (st.done[g]) {
    if (tid < W) st.parent[g * W + tid] = -1;
    return;
  }
  const long long c = st.count[g];
  if (c >= limit) {
    __syncthreads();  // every thread has read `done`
    if (tid == 0) st.done[g] = 2;
    if (tid < W) st.parent[g * W + tid] = -1;
    return;
  }
  for (int r = tid; r < K; r += ADV_THREADS) {
    const int32_t t = token[g * K + r];
    bool s = false;
    for (long long j = 0; j < n_stop; ++j) s = s || stop[j] == (uint32_t)t;
    is_stop[r] = s;
    cand_s[r] = score[g * K + r];
    cand_t[r] = t;
    cand_p[r] = parent[g * K + r];
  }
  for (int w = tid; w < W; w += ADV_THREADS) {
    fin_score[w] = st.fin_score[g * W + w];
    fin_len[w] = st.fin_len[g * W + w];
    src[w] = -1;
    new_par[w] = -1;
    new_cum[w] = neg_inf();
  }
  if ((tid & 31) == 0 && tid < 96)
    len_pow[tid >> 5] = pow((double)(tid == 0 ? c + 1 : tid == 32 ? c + 2 : limit), alpha);
  __syncthreads();
  if (tid == 0) {
    int live = 0, fins = st.fin_count[g];
    // slot of a hypothesis in the pool of the W best, or -1; equal lowest scores: the highest slot gives way
    auto insert = [&](float norm, int from, int len) {
      int slot = fins;
      if (fins >= W) {
        slot = 0;
        for (int w = 1; w < W; ++w)
          if (fin_score[w] <= fin_score[slot]) slot = w;
        if (!(norm > fin_score[slot])) return;
      } else {
        ++fins;
      }
      fin_score[slot] = norm;
      fin_len[slot] = len;
      src[slot] = from;
    };
    for (int r = 0; r < K; ++r) {
      if (cand_t[r] < 0 || cand_p[r] < 0 || cand_p[r] >= W) continue;
      if (is_stop[r]) {
        if (r < W) insert((float)((double)cand_s[r] / len_pow[0]), cand_p[r], (int)c);
      } else if (live < W) {
        new_par[live] = cand_p[r];
        new_tok[live] = cand_t[r];
        new_cum[live] = cand_s[r];
        ++live;
      }
    }
    int d = 0;
    if (c + 1 >= limit) {
      for (int w = 0; w < live; ++w) insert((float)((double)new_cum[w] / len_pow[0]), MAX_W + w, (int)c + 1);
      d = c + 1 >= max_seq_len ? 3 : 2;
    } else if (live == 0) {
      d = 1;
    } else if (fins >= W) {
      float low = fin_score[0], best = new_cum[0];
      for (int w = 1; w < W; ++w) {
        low = fminf(low, fin_score[w]);
        best = fmaxf(best, new_cum[w]);
      }
      const double ahead = fmax((double)best / len_pow[1], (double)best / len_pow[2]);
      if (early || (double)low >= ahead) d = 1;
    }
    live_n = live;
    fin_n = fins;
    code = d;
  }
  __syncthreads();
  int32_t* hist = st.tokens + g * W * st.cap;
  int32_t* fin = st.fin_tokens + g * W * st.cap;
  // hypotheses that ended in a stop token: their beam's tokens as they were
  for (int w = 0; w < W; ++w)
    if (src[w] >= 0 && src[w] < MAX_W)
      for (long long i = tid; i < c; i += ADV_THREADS) fin[w * st.cap + i] = hist[src[w] * st.cap + i];
  const int live = live_n;
  for (long long i0 = 0; i0 < c; i0 += ADV_THREADS) {
    const long long i = i0 + tid;
    if (i < c) {
      for (int w = 0; w < live; ++w) tile[w * ADV_THREADS + tid] = hist[new_par[w] * st.cap + i];
      for (int w = 0; w < live; ++w)
        if (new_par[w] != w) hist[w * st.cap + i] = tile[w * ADV_THREADS + tid];
    }
  }
  for (int w = tid; w < W; w += ADV_THREADS) {
    if (w < live) {
      hist[w * st.cap + c] = new_tok[w];
      st.last[g * W + w] = new_tok[w];
    }
    st.cum[g * W + w] = new_cum[w];
    st.parent[g * W + w] = new_par[w];
    st.fin_score[g * W + w] = fin_score[w];
    st.fin_len[g * W + w] = fin_len[w];
  }
  if (tid == 0) {
    st.count[g] = (int32_t)(c + 1);
    st.fin_count[g] = fin_n;
    st.done[g] = (uint8_t)code;
  }
  __syncthreads();
  // beams that reached the limit
  for (int w = 0; w < W; ++w)
    if (src[w] >= MAX_W)
      for (long long i = tid; i <= c; i += ADV_THREADS) fin[w * st.cap + i] = hist[(src[w] - MAX_W) * st.cap + i];
}

__global__ void __launch_bounds__(256) beam_reset_kernel(long long G, int W, BeamStatePtrs st) {
  const long long stride = (long long)gridDim.x * blockDim.x, me = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long n = G * W * st.cap;
  for (long long i = me; i < n; i += stride) {
    st.tokens[i] = 0;
    st.fin_tokens[i] = 0;
  }
  for (long long i = me; i < G * W; i += stride) {
    st.cum[i] = i % W == 0 ? 0.0f : neg_inf();
    st.last[i] = 0;
    st.parent[i] = -1;
    st.fin_len[i] = 0;
    st.fin_score[i] = neg_inf();
  }
  for (long long i = me; i < G; i += stride) {
    st.count[i] = 0;
    st.done[i] = 0;
    st.fin_count[i] = 0;
  }
}

// ---------------------------------------------------------------- reordering

constexpr int REORDER_MAX = 64;      // states of one launch
constexpr int REORDER_THREADS = 256;

struct ReorderState {
  const char* src;
  char* dst;
  long long src_row, dst_row;  // bytes between beams
  long long src_blk, dst_blk;  // bytes between the blocks of a beam
  long long vecs;              // vectors of a block
  long long tiles;             // tiles of a block
  long long blocks;
  long long first;             // first tile of the state in the launch
};

struct ReorderArgs {
  ReorderState s[REORDER_MAX];
  int n;
};

// A thread owns one vector position of all beams of a group: it reads every
// beam's new value before it writes one, so source and destination may be the
// same memory.  In place, beams that stay where they are are not touched.
template <typename Vec, int WB>
__global__ void __launch_bounds__(REORDER_THREADS) beam_reorder_kernel(const __grid_constant__ ReorderArgs a,
                                                                       const int32_t* __restrict__ parent, int W) {
  __shared__ int32_t par[WB];
  const long long tile = blockIdx.x;
  int k = 0;
  while (k + 1 < a.n && tile >= a.s[k + 1].first) ++k;
  const ReorderState& s = a.s[k];
  long long t = tile - s.first;
  const long long in_blk = t % s.tiles;
  t /= s.tiles;
  const long long blk = t % s.blocks, g = t / s.blocks;
  if (threadIdx.x < W) {
    const int32_t q = parent[g * W + threadIdx.x];
    par[threadIdx.x] = q >= 0 && q < W ? q : (int32_t)threadIdx.x;
  }
  __syncthreads();
  const long long i = in_blk * REORDER_THREADS + threadIdx.x;
  if (i >= s.vecs) return;
  const char* src = s.src + g * W * s.src_row + blk * s.src_blk + i * (long long)sizeof(Vec);
  char* dst = s.dst + g * W * s.dst_row + blk * s.dst_blk + i * (long long)sizeof(Vec);
  const bool same = s.src == s.dst;
  Vec v[WB];
#pragma unroll
  for (int w = 0; w < WB; ++w)
    if (w < W && !(same && par[w] == w)) v[w] = *(const Vec*)(src + par[w] * s.src_row);
#pragma unroll
  for (int w = 0; w < WB; ++w)
    if (w < W && !(same && par[w] == w)) *(Vec*)(dst + w * s.dst_row) = v[w];
}

}  // namespace pesti_rows
