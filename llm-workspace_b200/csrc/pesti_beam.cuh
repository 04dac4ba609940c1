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
//  beam_pick_kernel   a cluster of blocks per group, two, four or eight beams
//                     at a time in each.  For each beam, the K segments with the largest
//                     maxima hold the K largest logits: a team of warps finds
//                     them (a histogram of the maxima, its K-th place), reads
//                     them again and sorts what is above the K-th maximum,
//                     while another warp joins the row's sum.  The lists go to
//                     the first block's shared memory, which merges them.
//
// Accuracy of a row's log sum as the scan gives it, relative to the sum:
//   2^x by the hardware 2^-22.5; the rounding of x*c - R (one fused
//   operation): half an ulp of t = x*c - R, ln 2 * 2^-24 * E[|t|], and
//   E[|t|] <= 12 since the entropy of 2048 terms is at most 11 bits and R
//   less than 1 above the largest; c's own
//   rounding 1.34e-8 * E[m - x] (<= ln V <= 22); 16 additions in f32, 2^-24
//   each (units with NaN add in 64 bits).  Together below 1.95e-6.  (Beyond
//   |m*c| = 2^23 the rounding of m*c moves R by up to 32, but there logits lie
//   so far apart that nearly all mass has t of the largest: half an ulp of it
//   is at most 6.6e-7, within what c's rounding and the spread of t leave.)
//   Units are joined in 64 bits.  Two candidates of different beams whose
//   scores differ by less than twice LSE_EPS are therefore not ordered by these
//   sums: the merge adds up their rows again in 64 bits, in index order, and
//   ranks once more (random logits, 8 beams, K 16: about one group in 1500).
//   64-bit operations run at about 16 a cycle and SM, so rows are shared out
//   over the cluster where its blocks are not needed for other groups: two rows
//   add 33 us to a call of 32 groups of 8 x 152064 f32 (49 -> 82 us), eight 119.
//   In larger batches one block adds them up: two rows add 111 us to 64 groups
//   (76 -> 186 us), eight 430, and with more groups a call more often holds one.
#pragma once
#include "pesti_common.cuh"
#include "pesti_rowscan.cuh"

namespace pesti_rows {

constexpr int MAX_W = 64;          // beams of a group
constexpr int MAX_K = 128;         // candidates of a group
constexpr int SCAN_WARPS = 4;
constexpr int PICK_WARPS = 16;    // of a block: teams of TW warps, and a warp more for each
constexpr int MAX_PICK_CLUSTER = 8;
constexpr int MAX_SEL = MAX_K + MAX_K / 2 + 8;
constexpr int BINS = 256;
constexpr int RANK_CAP = 256;      // candidates that are ranked by counting
constexpr double LSE_EPS = 2e-6;
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

struct BeamWs {
  float2* unit;   // [rows][units] maximum and sum
  uint32_t* seg;  // [rows][units*8] order keys of the segment maxima
};

__device__ __forceinline__ bool beam_running(const float* cum, long long row) {
  return cum == nullptr || cum[row] > neg_inf();
}

// A warp a unit, bound by HBM where rows are many: 512 rows of 152064 f32 take
// 47.4 us, 6.6 TB/s; 256 rows of 128256 bf16, whose elements need twice the
// instructions a byte, 15.6 us, 4.2 TB/s (issue slots half used, 29 warps an SM);
// 4 rows of 32000 f32 4.4 us, a load's latency and the launch.  Blocks are
// small so that a finished warp's place is taken again soon.
template <typename T>
__global__ void __launch_bounds__(SCAN_WARPS * 32) beam_scan_kernel(const T* __restrict__ logits, long long ld,
                                                                    long long V, int W, long long units,
                                                                    long long blocks_per_row, const float* cum,
                                                                    const uint8_t* done, int every_row, BeamWs ws) {
  // the pick's blocks may start (and wait) once the last block here has started
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long row = blockIdx.x / blocks_per_row;
  const long long ub = blockIdx.x - row * blocks_per_row;
  const long long g = row / W;
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
    // eight chains of eight additions
    float2 a[4] = {};
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i) {
#pragma unroll
      for (int q = 0; q < Elem<T>::PAIRS; ++q) {
        float2 t = fma2(Elem<T>::pair(v[i], q), c2, r2);
        t.x = ex2(t.x);
        t.y = ex2(t.y);
        float2& to = a[(i * Elem<T>::PAIRS + q) & 3];
        to = add2(to, t);
      }
    }
    const float2 b = add2(add2(a[0], a[1]), add2(a[2], a[3]));
    S = warp_reduce_add(b.x + b.y);
  }
  if (far || S != S) {
    // the number of maxima, or a sum that leaves NaN out (one chain of 32 or 64 terms a lane, so in 64 bits)
    double s = 0.0;
#pragma unroll 1
    for (int i = 0; i < UNIT_VECS; ++i) {
      const uint4 w = i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : i == 3 ? v[3] : i == 4 ? v[4] : i == 5 ? v[5] : i == 6 ? v[6] : v[7];
      for (int q = 0; q < Elem<T>::PAIRS; ++q) {
        const float2 x = Elem<T>::pair(w, q);
        if (far) {
          s += (x.x == m ? 1.0 : 0.0) + (x.y == m ? 1.0 : 0.0);
        } else {
          if (x.x == x.x) s += (double)ex2(fmaf(x.x, LOG2E_F, -R));
          if (x.y == x.y) s += (double)ex2(fmaf(x.y, LOG2E_F, -R));
        }
      }
    }
    S = (float)warp_reduce_add(s);
  }
  if (lane < UNIT_VECS) {
    const bool none = !(mine > neg_inf());
    ws.seg[(row * units + u) * UNIT_VECS + lane] = none ? KEY_NEG_INF : order_key(mine);
  }
  if (lane == 0) ws.unit[row * units + u] = make_float2(m, S);
}

// A block of a group's cluster: `teams` teams of TW warps that select for beams
// first, first + 1, ... of the block's `rows`, then as many warps that join
// sums.  A team's arrays lie in dynamic shared memory behind the x and idx of
// the group's lists; the merge's scores take their place.
struct PickPlan {
  // nkeys: a multiple of 4; run: segments of a key; cap: entries of a team's list
  int W, K, rows, teams, nkeys, run, cap;
  int stay;  // the cluster's blocks help to add up rows again
  long long units;
};

template <int TW>
struct Team {
  int id, tid;                    // team, thread of the team
  uint32_t* keys;                 // [nkeys]
  unsigned long long* list;       // [cap] key << 32 | ~index
  int* hist;                      // [BINS]
  int* sel;                       // [MAX_SEL]
  int* word;                      // 32 words, below
  int turn;
};
enum { TM_NSEL = 0, TM_NLIST = 1, TM_OVER = 2, TM_T = 3, TM_MAX = 4, TM_MIN = 5, TM_CUT = 6, TM_COUNT = 8 };  // COUNT: 2 x 8

constexpr int TEAM_WORDS = BINS + MAX_SEL + 32;

// The block's dynamic shared memory: the lists, then for every team its list, keys and words (the histogram first).
__host__ __device__ __forceinline__ long long list_bytes(int W, int K) { return ((long long)W * K * 8 + 15) / 16 * 16; }
__host__ __device__ __forceinline__ long long keys_offset(int cap) { return (long long)cap * 8; }
__host__ __device__ __forceinline__ long long hist_offset(int nkeys, int cap) {
  return keys_offset(cap) + (long long)nkeys * 4;
}
__host__ __device__ __forceinline__ long long team_bytes(int nkeys, int cap) {
  return (hist_offset(nkeys, cap) + TEAM_WORDS * 4 + 15) / 16 * 16;
}

template <int TW>
__device__ __forceinline__ void team_sync(const Team<TW>& t) {
  if (TW == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(t.id + 1), "n"(TW * 32) : "memory");
}

// Sum over the team of one count per thread.
template <int TW>
__device__ __forceinline__ int team_count(Team<TW>& t, int c) {
  const int s = __reduce_add_sync(FULL, c);
  if (TW == 1) return s;
  int* buf = t.word + TM_COUNT + t.turn * 8;
  t.turn ^= 1;
  if ((t.tid & 31) == 0) buf[t.tid >> 5] = s;
  team_sync(t);
  int r = 0;
#pragma unroll
  for (int i = 0; i < TW; ++i) r += buf[i];
  return r;
}

// Appends a vector's elements >= cut to the team's list (OVER is set if they do not fit).
template <typename T, int TW>
__device__ __forceinline__ void append_vec(const Team<TW>& t, int cap, const uint4& v, long long first, float cut) {
  uint32_t in = 0;
#pragma unroll
  for (int q = 0; q < Elem<T>::PAIRS; ++q) {
    const float2 x = Elem<T>::pair(v, q);
    in |= (x.x >= cut ? 1u : 0u) << (2 * q) | (x.y >= cut ? 2u : 0u) << (2 * q);
  }
  while (in) {
    const int e = __ffs(in) - 1;
    in &= in - 1;
    const int at = atomicAdd(t.word + TM_NLIST, 1);
    if (at < cap)
      t.list[at] = ((unsigned long long)order_key(Elem<T>::at(v, e)) << 32) | (uint32_t)~(uint32_t)(first + e);
    else
      t.word[TM_OVER] = 1;
  }
}

template <typename T>
__device__ __forceinline__ uint4 load_seg_vec(const T* p, int head, long long V, long long seg, int lane) {
  const long long first = (seg * 32 + lane) * Elem<T>::VE - head;
  if (first >= 0 && first + Elem<T>::VE <= V) return __ldg((const uint4*)(p - head) + seg * 32 + lane);
  return load_edge<T>(p, first, V);
}

// (Everything is inlined: a call that takes the team would put it in local
// memory, and its arrays out of the compiler's sight as shared memory; 64 groups
// of 8: 22 us with calls.)

// Cuts the list to its largest entries, at least K and at most RANK_CAP (entries are distinct).
template <int TW>
__device__ __forceinline__ void prune_list(Team<TW>& t, int K) {
  constexpr int N = TW * 32, PER = (RANK_CAP + TW * 256 + N - 1) / N;
  team_sync(t);
  const int n = t.word[TM_NLIST];
  team_sync(t);  // every thread has read it before the next append (and left the last count's buffer)
  if (n <= RANK_CAP) return;
  unsigned long long lo = 0, hi = ~0ull;
  while (hi - lo > 1) {
    const unsigned long long mid = lo + (hi - lo) / 2;
    int c = 0;
    for (int i = t.tid; i < n; i += N) c += t.list[i] >= mid;
    c = team_count(t, c);
    if (c >= K) {
      lo = mid;
      if (c <= RANK_CAP) break;
    } else {
      hi = mid;
    }
  }
  // entries kept move to the front; each thread holds its own first
  unsigned long long mine[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = t.tid + j * N;
    mine[j] = i < n ? t.list[i] : 0ull;
  }
  team_sync(t);
  if (t.tid == 0) t.word[TM_NLIST] = 0;
  team_sync(t);
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (mine[j] != 0ull && mine[j] >= lo) t.list[atomicAdd(t.word + TM_NLIST, 1)] = mine[j];
  team_sync(t);
}

// The least key of the segments to read, by bisection, and those segments:
// for maxima that the histogram does not tell apart.
template <int TW>
__device__ __forceinline__ uint32_t select_by_bisection(Team<TW>& t, int nkeys, int K, uint32_t kmax, int most) {
  constexpr int N = TW * 32;
  uint32_t lo = KEY_NEG_INF + 1, hi = kmax + 1;
  int above = most + 1;
  while (hi - lo > 1 && above > most) {
    const uint32_t mid = lo + (hi - lo) / 2;
    int c = 0;
    for (int i = t.tid; i < nkeys; i += N) c += t.keys[i] >= mid;
    c = team_count(t, c);
    if (c >= K) {
      lo = mid;
      above = c;
    } else {
      hi = mid;
    }
  }
  if (above <= most) {
    for (int i = t.tid; i < nkeys; i += N)
      if (t.keys[i] >= lo) t.sel[atomicAdd(t.word + TM_NSEL, 1)] = i;
  } else {
    // many segments share the K-th maximum: those above it, then the first ones at it
    int c = 0;
    for (int i = t.tid; i < nkeys; i += N) c += t.keys[i] > lo;
    const int over = team_count(t, c);
    if (t.tid < 32) {
      int left = K - over;
      for (int i0 = 0; i0 < nkeys; i0 += 32) {
        const int i = i0 + t.tid;
        const uint32_t k = i < nkeys ? t.keys[i] : 0u;
        const uint32_t same = __ballot_sync(FULL, k == lo);
        const int before = __popc(same & ((1u << t.tid) - 1u));
        if (k > lo || (k == lo && before < left)) t.sel[atomicAdd(t.word + TM_NSEL, 1)] = i;
        left -= min(left, __popc(same));
      }
    }
  }
  team_sync(t);
  return lo;
}

// The first bin whose running count reaches K goes to CUT, -1 if there is none or the count is above `most`.
// In step before (the bins are filled) and behind it.
template <int TW>
__device__ __forceinline__ void find_bin(const Team<TW>& t, int K, int most) {
  if (t.tid < 32) {
    // lane l adds up bins 8l..8l+7
    const int4 c0 = ((const int4*)t.hist)[2 * t.tid], c1 = ((const int4*)t.hist)[2 * t.tid + 1];
    const int sum = c0.x + c0.y + c0.z + c0.w + c1.x + c1.y + c1.z + c1.w;
    int upto = warp_incl_scan_add(sum);
    const uint32_t hit = __ballot_sync(FULL, upto >= K);
    if (hit == 0) {
      if (t.tid == 0) t.word[TM_CUT] = -1;
    } else if (t.tid == __ffs(hit) - 1) {
      upto -= sum;
      int bin = 8 * t.tid - 1;
      while (upto < K) upto += t.hist[++bin];
      t.word[TM_CUT] = upto <= most ? bin : -1;
    }
  }
  team_sync(t);
}

// Segment i of the selected ones (WIDE: runs of segments).
template <bool WIDE, int TW>
__device__ __forceinline__ long long selected(const Team<TW>& t, const PickPlan& pl, int i) {
  return WIDE ? (long long)t.sel[i / pl.run] * pl.run + i % pl.run : (long long)t.sel[i];
}

// The elements of the selected segments in rounds that keep the list short.
template <typename T, int TW, bool WIDE>
__device__ __forceinline__ void append_in_rounds(Team<TW>& t, const PickPlan& pl, const T* p, long long V, int todo,
                                                 float cut) {
  const int lane = t.tid & 31, head = row_head<T>(p);
  team_sync(t);
  if (t.tid == 0) t.word[TM_NLIST] = 0;
  team_sync(t);
  for (int i0 = 0; i0 < todo; i0 += TW) {
    const int i = i0 + (t.tid >> 5);
    if (i < todo) {
      const long long sg = selected<WIDE>(t, pl, i);
      const uint4 v = load_seg_vec<T>(p, head, V, sg, lane);
      // at most TW * 256 behind at most RANK_CAP
      append_vec<T, TW>(t, pl.cap, v, (sg * 32 + lane) * Elem<T>::VE - head, cut);
    }
    prune_list(t, pl.K);
  }
}

// The K largest logits of a row, in order, to x and idx; returns their number.
// Nearly all of this runs once: its time is instruction fetches and the
// latency of two dependent reads, so loops stay rolled unless they load.
template <typename T, int TW, bool WIDE>
__device__ __forceinline__ int pick_row(Team<TW>& t, const PickPlan& pl, const T* p, long long V, const uint32_t* seg,
                                        float* xs, int32_t* ids) {
  constexpr int N = TW * 32;
  const int lane = t.tid & 31, K = pl.K, nkeys = pl.nkeys;
  if (WIDE) {
    const long long nseg = pl.units * UNIT_VECS;
    for (int i = t.tid; i < nkeys; i += N) {
      uint32_t k = KEY_NEG_INF;
      const long long end = min(nseg, (long long)(i + 1) * pl.run);
      for (long long j = (long long)i * pl.run; j < end; ++j) k = max(k, seg[j]);
      t.keys[i] = k;
    }
  } else {
    // 16 keys of a thread in flight at once (their number is a multiple of 8)
    for (int i0 = t.tid * 4; i0 < nkeys; i0 += N * 16) {
      uint4 k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j * N * 4 < nkeys) k[j] = *(const uint4*)(seg + i0 + j * N * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j * N * 4 < nkeys) *(uint4*)(t.keys + i0 + j * N * 4) = k[j];
    }
  }
  for (int i = t.tid; i < BINS; i += N) t.hist[i] = 0;
  if (t.tid < TM_COUNT)
    t.word[t.tid] = t.tid == TM_T || t.tid == TM_MIN ? (int)0xffffffffu : 0;
  team_sync(t);
  uint32_t kmax = KEY_NEG_INF, kmin = 0xffffffffu;
  int valid = 0;
#pragma unroll 2
  for (int i = t.tid; i < nkeys; i += N) {
    const uint32_t k = t.keys[i];
    const bool v = k > KEY_NEG_INF;
    valid += v;
    kmin = min(kmin, v ? k : 0xffffffffu);
    kmax = max(kmax, k);
  }
  kmax = __reduce_max_sync(FULL, kmax);
  kmin = __reduce_min_sync(FULL, kmin);
  if (lane == 0) {
    atomicMax((uint32_t*)t.word + TM_MAX, kmax);
    atomicMin((uint32_t*)t.word + TM_MIN, kmin);
  }
  valid = team_count(t, valid);
  kmax = (uint32_t)t.word[TM_MAX];
  kmin = (uint32_t)t.word[TM_MIN];
  if (valid == 0) return 0;
  const int most = K + K / 2 + 8;
  bool binned = valid > K && kmax != kmin;
  uint32_t least = KEY_NEG_INF + 1;
  const bool whole = valid <= K || (valid <= most && kmax == kmin);  // every segment with a finite value
  if (whole) {
    for (int i = t.tid; i < nkeys; i += N)
      if (t.keys[i] > KEY_NEG_INF) t.sel[atomicAdd(t.word + TM_NSEL, 1)] = i;
    if (valid >= K) least = kmin;
  }
  if (binned) {
    // 256 bins of equal width of the keys, from the largest down (over four powers of two at most)
    const int sh = max(0, 24 - __clz((int)min(kmax - kmin, 0x1ffffffu)));
#pragma unroll 2
    for (int i = t.tid; i < nkeys; i += N) {
      const uint32_t b = (kmax - t.keys[i]) >> sh;
      if (b < BINS) atomicAdd(t.hist + b, 1);
    }
    team_sync(t);
    find_bin(t, K, most);
    const int bin = t.word[TM_CUT];
    binned = bin >= 0;
    if (binned) {
      least = 0xffffffffu;
#pragma unroll 2
      for (int i = t.tid; i < nkeys; i += N) {
        const uint32_t k = t.keys[i];
        if ((kmax - k) >> sh <= (uint32_t)bin) {
          t.sel[atomicAdd(t.word + TM_NSEL, 1)] = i;
          least = min(least, k);
        }
      }
      least = __reduce_min_sync(FULL, least);
    }
  }
  if (!whole && !binned) least = select_by_bisection(t, nkeys, K, kmax, most);
  if (lane == 0) atomicMin((uint32_t*)t.word + TM_T, least);
  team_sync(t);
  float cut = key_value((uint32_t)t.word[TM_T]);
  // their elements from the cut up: all at once, or in rounds that keep the list short
  const int todo = t.word[TM_NSEL] * (WIDE ? pl.run : 1), head = row_head<T>(p);
  if (valid < K) {
    // fewer segments than K say nothing of the K-th logit: the maxima of their vectors do
    for (int i = t.tid; i < BINS; i += N) t.hist[i] = 0;
    team_sync(t);
    constexpr int sh = 17;  // 64 bins to a power of two
#pragma unroll 2
    for (int i = t.tid >> 5; i < todo; i += TW) {
      const float m = Elem<T>::vec_max(load_seg_vec<T>(p, head, V, selected<WIDE>(t, pl, i), lane));
      const uint32_t b = (kmax - order_key(m)) >> sh;
      if (m > neg_inf() && b < BINS) atomicAdd(t.hist + b, 1);
    }
    team_sync(t);
    find_bin(t, K, 0x7fffffff);
    const int bin = t.word[TM_CUT];
    const uint32_t down = ((uint32_t)bin + 1u) << sh;
    if (bin >= 0 && down < kmax - KEY_NEG_INF) cut = key_value(kmax - down + 1u);
  }
  for (int i0 = t.tid >> 5; i0 < todo; i0 += 8 * TW) {
    uint4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * TW < todo) v[j] = load_seg_vec<T>(p, head, V, selected<WIDE>(t, pl, i0 + j * TW), lane);
    uint32_t in = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * TW < todo) in |= (Elem<T>::vec_max(v[j]) >= cut ? 1u : 0u) << j;
    while (in) {
      const int j = __ffs(in) - 1;
      in &= in - 1;
      uint4 w = v[0];
#pragma unroll
      for (int q = 1; q < 8; ++q)
        if (q == j) w = v[q];
      append_vec<T, TW>(t, pl.cap, w, (selected<WIDE>(t, pl, i0 + j * TW) * 32 + lane) * Elem<T>::VE - head, cut);
    }
  }
  team_sync(t);
  if (t.word[TM_OVER]) append_in_rounds<T, TW, WIDE>(t, pl, p, V, todo, cut);
  if (t.word[TM_NLIST] > RANK_CAP) prune_list(t, K);
  const int nl = t.word[TM_NLIST];
  int tops = 0;
  for (int i = t.tid; i < nl; i += N) {
    const unsigned long long c = t.list[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < nl; ++j) rank += t.list[j] > c;
    if (rank < K) {
      xs[rank] = key_value((uint32_t)(c >> 32));
      ids[rank] = (int32_t)~(uint32_t)c;
    }
    tops += (uint32_t)(c >> 32) == 0xff800000u;  // +inf
  }
  int n = min(nl, K);
  // a row's +inf entries share its probability; the others have none
  if (kmax == 0xff800000u) n = min(n, team_count(t, tops));
  return n;
}

struct PickShared {
  double ref[MAX_W], logs[MAX_W], cum[MAX_W];  // logp(x) = (x - ref) - logs, or -logs for x = ref = +inf
  double red[40];
  int n[MAX_W];
  int sorted[RANK_CAP], reach[RANK_CAP];
  int part[MAX_W], part_at[MAX_W];
  double pow2[256];  // 2^(i/256)
  double again[MAX_W][MAX_PICK_CLUSTER];
  int ranked;
  unsigned long long next;  // the best score that is not among the ranked (0: none)
  unsigned long long flagged;
};

// e^d for d <= 0 (0 below -700, and for NaN), within 2^-51: a table of 2^(i/256) and a polynomial on |r| <= ln 2 / 512
// (P. T. P. Tang's table-driven method, ACM Trans. Math. Softw. 15, 1989; r^5/120 is below 2^-54).  A row's sum is
// bound by the rate of 64-bit operations: 12 of them a logit.
__device__ __forceinline__ double exp_by_table(const double* pow2, double d) {
  // 256 / ln 2, and ln 2 / 256 in two parts, the first of 29 bits
  constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the rounded integer
  const double t = fma(d, 369.3299304675746, MAGIC);
  const int n = __double2loint(t);
  const double k = t - MAGIC;
  const double r = fma(k, -0x1.f473de6af278fp-38, fma(k, -0x1.62e42fe000000p-9, d));
  const double y = fma(r * r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), r);
  const double e = pow2[n & 255];
  const double v = fma(e, y, e);
  return d >= -700.0 ? __hiloint2double(__double2hiint(v) + ((n >> 8) << 20), __double2loint(v)) : 0.0;
}

__device__ __forceinline__ double beam_score(const PickShared& sh, int w, float x) {
  return sh.ref[w] == (double)pos_inf() ? sh.cum[w] - sh.logs[w] : sh.cum[w] + (((double)x - sh.ref[w]) - sh.logs[w]);
}

// Order-preserving image of a double (no NaN), and back.
__device__ __forceinline__ unsigned long long order_key64(double d) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(d + 0.0);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value64(unsigned long long k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
}

// Ranks the candidates of the group's lists; `sorted` gets the positions
// w * K + r of the first min(ranked, RANK_CAP) (K at least, if there are as
// many).  Returns the number of candidates.
__device__ __forceinline__ int rank_candidates(PickShared& sh, const float* xs, unsigned long long* score, int W, int K) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int total = 0;
  for (int w = 0; w < W; ++w) total += sh.n[w];
  const int all = W * K;
  for (int j = threadIdx.x; j < all; j += blockDim.x) {
    const int w = j / K;
    score[j] = j - w * K < sh.n[w] ? order_key64(beam_score(sh, w, xs[j])) : 0ull;
  }
  __syncthreads();
  if (all <= RANK_CAP) {
    // a warp per candidate: those ahead are larger, or equal and of a lower beam (or earlier in the list)
    for (int j = wid; j < all; j += warps) {
      const unsigned long long s = score[j];
      int rank = 0;
      for (int o = lane; o < all; o += 32) rank += score[o] + (o < j) > s;
      rank = __reduce_add_sync(FULL, rank);
      if (lane == 0 && s != 0ull) sh.sorted[rank] = j;
    }
    if (threadIdx.x == 0) {
      sh.ranked = total;
      sh.next = 0ull;
    }
    __syncthreads();
    return total;
  }
  if (wid == 0) {
    // a score that between K and RANK_CAP candidates reach: lane l counts in the (sorted) lists l and l + 32
    auto count = [&](unsigned long long t, int w) {
      int lo = 0, hi = w < W ? sh.n[w] : 0;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (score[w * K + mid] >= t)
          lo = mid + 1;
        else
          hi = mid;
      }
      return lo;
    };
    unsigned long long lo = 1ull, hi = ~0ull;
    int have = total;
    while (have > RANK_CAP && hi - lo > 1) {
      const unsigned long long mid = lo + (hi - lo) / 2;
      const int c = __reduce_add_sync(FULL, count(mid, lane) + count(mid, lane + 32));
      if (c >= K) {
        lo = mid;
        have = c;
      } else {
        hi = mid;
      }
    }
    // the lists' parts that reach it, one behind the other
    const int a = count(lo, lane), b = count(lo, lane + 32);
    const int at_a = warp_incl_scan_add(a) - a, first = __reduce_add_sync(FULL, a);
    const int at_b = first + warp_incl_scan_add(b) - b;
    sh.part[lane] = a;
    sh.part[lane + 32] = b;
    sh.part_at[lane] = at_a;
    sh.part_at[lane + 32] = at_b;
    // the best of the lists' rests; where too many share one score, that score itself
    auto rest = [&](int w, int n) { return w < W && n < sh.n[w] ? score[w * K + n] : 0ull; };
    unsigned long long next = max(rest(lane, a), rest(lane + 32, b));
    const uint32_t high = __reduce_max_sync(FULL, (uint32_t)(next >> 32));
    const uint32_t low = __reduce_max_sync(FULL, (uint32_t)(next >> 32) == high ? (uint32_t)next : 0u);
    next = ((unsigned long long)high << 32) | low;
    if (lane == 0) {
      sh.ranked = have;
      sh.next = have <= RANK_CAP ? next : lo;
    }
  }
  __syncthreads();
  const int have = sh.ranked;
  if (have <= RANK_CAP) {
    for (int j = threadIdx.x; j < all; j += blockDim.x) {
      const int w = j / K, r = j - w * K;
      if (r < sh.part[w]) sh.reach[sh.part_at[w] + r] = j;
    }
    __syncthreads();
    for (int i = wid; i < have; i += warps) {
      const int j = sh.reach[i];
      const unsigned long long s = score[j];
      int rank = 0;
      for (int o = lane; o < have; o += 32) rank += score[sh.reach[o]] + (o < i) > s;
      rank = __reduce_add_sync(FULL, rank);
      if (lane == 0) sh.sorted[rank] = j;
    }
    __syncthreads();
    return total;
  }
  // more than RANK_CAP candidates share the K-th score: by bisection in every list
  for (int j = threadIdx.x; j < all; j += blockDim.x) {
    const unsigned long long s = score[j];
    if (s == 0ull) continue;
    const int w = j / K;
    int rank = j - w * K;
    for (int o = 0; o < W && rank < RANK_CAP; ++o) {
      if (o == w) continue;
      int lo = 0, hi = sh.n[o];
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (score[o * K + mid] >= s + (o > w))
          lo = mid + 1;
        else
          hi = mid;
      }
      rank += lo;
    }
    if (rank < RANK_CAP) sh.sorted[rank] = j;
  }
  __syncthreads();
  return total;
}

// The address of a shared variable of another block of the cluster.
template <typename P>
__device__ __forceinline__ P* in_block(P* p, uint32_t rank) {
  unsigned long long r;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"((unsigned long long)p), "r"(rank));
  return (P*)r;
}

// Bound by latency: dependent reads (keys, segments), the steps between them
// and their first instruction fetches.  9.3 us for one group of 4 beams x 32000
// f32, 13.4 us for 32 groups of 8 x 128256 bf16, 13.0 us for 64 groups of 8 x
// 152064 f32, a few of which the scan's end hides.
template <typename T, int TW, bool WIDE>
__global__ void __launch_bounds__(PICK_WARPS * 32) beam_pick_kernel(
    const T* __restrict__ logits, long long ld, long long V, const __grid_constant__ PickPlan pl, const float* cum,
    const uint8_t* done, BeamWs ws, float* out_score, int32_t* out_token, int32_t* out_parent, float* out_lse) {
  extern __shared__ __align__(16) char dyn[];
  __shared__ PickShared sh;
  const int tid = threadIdx.x, lane = tid & 31, W = pl.W, K = pl.K;
  uint32_t csize, crank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
  // every block of the cluster has begun before anything is written to the first one
  if (csize > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  const long long g = blockIdx.x / csize, row0 = g * W;
  float* xs = (float*)dyn;
  int32_t* ids = (int32_t*)(xs + W * K);
  char* teams = dyn + list_bytes(W, K);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (csize > 1) asm volatile("barrier.cluster.wait;" ::: "memory");

  const bool group_done = done && done[g];
  const int wid = tid >> 5, from = (int)crank * pl.rows, to = min(W, from + pl.rows);
  PickShared* first = csize > 1 ? in_block(&sh, 0) : &sh;
  if (wid < pl.teams * TW) {
    Team<TW> t;
    t.id = wid / TW;
    t.tid = tid - t.id * TW * 32;
    t.turn = 0;
    char* const mine = teams + t.id * team_bytes(pl.nkeys, pl.cap);
    t.list = (unsigned long long*)mine;
    t.keys = (uint32_t*)(mine + keys_offset(pl.cap));
    t.hist = (int*)(mine + hist_offset(pl.nkeys, pl.cap));
    t.sel = t.hist + BINS;
    t.word = t.sel + MAX_SEL;
    float* const first_xs = csize > 1 ? in_block(xs, 0) : xs;
    int32_t* const first_ids = csize > 1 ? in_block(ids, 0) : ids;
    for (int w = from + t.id; w < to; w += pl.teams) {
      int n = 0;
      if (!group_done && beam_running(cum, row0 + w))
        n = pick_row<T, TW, WIDE>(t, pl, logits + (row0 + w) * ld, V, ws.seg + (row0 + w) * pl.units * UNIT_VECS,
                                  first_xs + w * K, first_ids + w * K);
      if (t.tid == 0) first->n[w] = n;
      team_sync(t);
    }
  } else {
    for (int w = from + wid - pl.teams * TW; w < to; w += pl.teams) {
      // the row's sum, joined from its units in a fixed order
      const long long row = row0 + w;
      double ref = 0.0, logs = 0.0;
      if (!group_done && (out_lse || beam_running(cum, row))) {
        const float2* unit = ws.unit + row * pl.units;
        float m = neg_inf();
        for (long long u = lane; u < pl.units; u += 32) m = fmaxf(m, unit[u].x);
        m = warp_max(m);
        if (m > neg_inf()) {
          double s = 0.0;
          for (long long u = lane; u < pl.units; u += 32) {
            const float2 a = unit[u];
            if (a.x > neg_inf()) s += (double)a.y * ref_scale(a.x, m, LOG2E_F);
          }
          s = warp_reduce_add(s);
          // sum 2^(x c - R) = 2^(m c - R) sum 2^((x - m) c)
          ref = (double)m;
          logs = is_far(m, LOG2E_F) ? log(s)
                                    : LN2 * (log2(s) - ((double)m * (double)LOG2E_F - (double)ceilf(m * LOG2E_F)));
        }
        if (out_lse && lane == 0) out_lse[row] = m > neg_inf() ? (float)(ref + (m < pos_inf() ? logs : 0.0)) : m;
      } else if (out_lse && lane == 0) {
        out_lse[row] = neg_inf();
      }
      if (lane == 0) {
        first->ref[w] = ref;
        first->logs[w] = logs;
        first->cum[w] = cum ? (double)cum[row] : 0.0;
      }
    }
  }
  if (csize > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    if (crank != 0 && !pl.stay) return;
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
  const uint32_t parts = pl.stay ? csize : 1u;  // blocks that add up rows again
  __syncthreads();
  unsigned long long* score = (unsigned long long*)teams;
  int total = 0;
  unsigned long long flagged = 0ull;
  if (crank == 0) {
    total = rank_candidates(sh, xs, score, W, K);
    const int have = min(sh.ranked, RANK_CAP);
    if (wid == 0) {
      // neighbours whose order the sums do not settle, up to the first clear gap behind the K-th place
      uint32_t lo = 0, hi = 0;
      bool open = W > 1;
      for (int i0 = 0; open && i0 < have; i0 += 32) {
        const int i = i0 + lane;
        bool near = false;
        int wa = 0, wb = 0;
        // the last of the ranked is compared with the best behind them
        if (i + 1 < have || (i + 1 == have && sh.next != 0ull)) {
          const bool last = i + 1 == have;
          const int ja = sh.sorted[i], jb = last ? ja : sh.sorted[i + 1];
          const double a = key_value64(score[ja]), b = key_value64(last ? sh.next : score[jb]);
          near = !(a - b > 2.0 * LSE_EPS) && a < (double)pos_inf();
          wa = ja / K;
          wb = jb / K;
        }
        const uint32_t gap = __ballot_sync(FULL, !near && i >= K - 1 && i < have);
        open = gap == 0;
        if (near && wa != wb && (open || lane < __ffs(gap) - 1)) {
          const unsigned long long both = (1ull << wa) | (1ull << wb);
          lo |= (uint32_t)both;
          hi |= (uint32_t)(both >> 32);
        }
      }
      lo = __reduce_or_sync(FULL, lo);
      hi = __reduce_or_sync(FULL, hi);
      if (open && total > have) {
        // a run that leaves the ranked part: every row with candidates (the others may not be read)
        lo = __ballot_sync(FULL, lane < W && sh.n[lane] > 0);
        hi = __ballot_sync(FULL, lane + 32 < W && sh.n[lane + 32] > 0);
      }
      // the blocks that stayed are told
      flagged = ((unsigned long long)hi << 32) | lo;
      if (lane > 0 && lane < parts) *in_block(&sh.flagged, lane) = flagged;
      if (flagged)
        for (uint32_t r = 1; r < parts; ++r)
          for (int w = lane; w < W; w += 32) *in_block(&sh.ref[w], r) = sh.ref[w];
      if (lane == 0) sh.flagged = flagged;
    }
  }
  if (parts > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    if (crank != 0) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
  __syncthreads();
  flagged = sh.flagged;
  if (flagged) {
    if (parts > 1 && crank == 0) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    for (int i = tid; i < 256; i += blockDim.x) sh.pow2[i] = exp2((double)i / 256.0);
    __syncthreads();
    // each block its part of every row; the parts are as long for every row, and joined in order
    const long long part = (V + parts - 1) / parts, begin = crank * part, stop = min(V, begin + part);
    for (int w = 0; w < W; ++w) {
      if (!((flagged >> w) & 1ull) || sh.ref[w] == (double)pos_inf()) continue;
      const T* q = logits + (row0 + w) * ld;
      const double m = sh.ref[w];
      double s = 0.0;
      // 16 logits of a thread in flight
      for (long long v0 = begin + tid; v0 < stop; v0 += 16 * blockDim.x) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const long long v = v0 + i * (long long)blockDim.x;
          x[i] = v < stop ? Elem<T>::load(q, v) : neg_inf();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s += exp_by_table(sh.pow2, (double)x[i] - m);
      }
      s = block_reduce_add(s, sh.red);
      if (tid == 0) first->again[w][crank] = s;
    }
    if (parts > 1) {
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      if (crank != 0) return;
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    __syncthreads();
    for (int w = tid; w < W; w += blockDim.x)
      if (((flagged >> w) & 1ull) && sh.ref[w] != (double)pos_inf()) {
        double s = 0.0;
        for (uint32_t r = 0; r < parts; ++r) s += sh.again[w][r];
        sh.logs[w] = log(s);
      }
    __syncthreads();
    rank_candidates(sh, xs, score, W, K);
  }
  if (crank != 0) return;
  for (int r = tid; r < K; r += blockDim.x) {
    float sc = neg_inf();
    int tk = -1, pa = -1;
    if (r < total) {
      const int j = sh.sorted[r];
      pa = j / K;
      sc = (float)key_value64(score[j]);
      tk = ids[j];
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

// One block per group.  One warp walks over the ranks, the pool's scores in its
// lanes: which candidates end, which go on, and which slots of the pool they
// take.  The block then moves the token histories: a thread owns a column of
// all beams, so rows exchange places without another buffer.  A step's time is
// three dependent reads and the ranks, some 60 cycles each: 4.6 us for 4 beams
// and 8 candidates, 9.2 us for 128 groups of 8 and 16 (steps of a captured
// search; the bytes moved are some KB a group).
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
  __shared__ float new_cum[MAX_W];
  __shared__ int32_t src[MAX_W], new_par[MAX_W], new_tok[MAX_W];
  __shared__ double len_pow[3];
  __shared__ int live_n;
  static_assert(MAX_W == 64 && ADV_THREADS >= MAX_K, "two pool slots a lane, a thread per candidate");
  const long long g = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const long long limit = min(max_tokens, max_seq_len);
  // everything a step needs is on its way at once
  const uint8_t was_done = st.done[g];
  const long long c = st.count[g];
  const int had = st.fin_count[g];
  if (tid < K) {
    const int32_t t = token[g * K + tid];
    cand_s[tid] = score[g * K + tid];
    cand_p[tid] = parent[g * K + tid];
    cand_t[tid] = t;
    bool s = false;
    for (long long j = 0; j < n_stop; ++j) s = s || stop[j] == (uint32_t)t;
    is_stop[tid] = s;
  }
  if (tid < W) {
    src[tid] = -1;
    new_par[tid] = -1;
    new_cum[tid] = neg_inf();
  }
  // the pool: slots lane and lane + 32; slots that are not there never have the lowest score
  float fin0 = pos_inf(), fin1 = pos_inf();
  int len0 = 0, len1 = 0;
  if (tid < 32) {
    if (lane < W) {
      fin0 = st.fin_score[g * W + lane];
      len0 = st.fin_len[g * W + lane];
    }
    if (lane + 32 < W) {
      fin1 = st.fin_score[g * W + lane + 32];
      len1 = st.fin_len[g * W + lane + 32];
    }
  }
  if (was_done || c >= limit) {
    __syncthreads();  // every thread has read `done`
    if (tid == 0 && !was_done) st.done[g] = c >= max_seq_len ? 3 : 2;
    if (tid < W) st.parent[g * W + tid] = -1;
    return;
  }
  if (lane == 0 && tid >= 32 && tid < 128)
    len_pow[(tid >> 5) - 1] = pow((double)(tid == 32 ? c + 1 : tid == 64 ? c + 2 : limit), alpha);
  __syncthreads();
  if (tid < 32) {
    int live = 0, fins = had;
    // a hypothesis goes to the pool of the W best; of equal lowest scores the highest slot gives way
    auto lowest = [&](uint32_t& low) {
      const uint32_t k0 = lane < W ? order_key(fin0) : 0xffffffffu, k1 = lane + 32 < W ? order_key(fin1) : 0xffffffffu;
      low = __reduce_min_sync(FULL, min(k0, k1));
      const uint32_t in1 = __ballot_sync(FULL, k1 == low), in0 = __ballot_sync(FULL, k0 == low);
      return in1 ? 63 - __clz(in1) : 31 - __clz(in0);
    };
    auto insert = [&](float norm, int from, int len) {
      int slot = fins;
      if (fins >= W) {
        uint32_t low;
        slot = lowest(low);
        if (!(norm > key_value(low))) return;
      } else {
        ++fins;
      }
      if (slot == lane) {
        fin0 = norm;
        len0 = len;
      }
      if (slot == lane + 32) {
        fin1 = norm;
        len1 = len;
      }
      if (lane == 0) src[slot] = from;
    };
    for (int r = 0; r < K; ++r) {
      const int t = cand_t[r], q = cand_p[r];
      if (t < 0 || q < 0 || q >= W) continue;
      if (is_stop[r]) {
        if (r < W) insert((float)((double)cand_s[r] / len_pow[0]), q, (int)c);
      } else if (live < W) {
        if (lane == 0) {
          new_par[live] = q;
          new_tok[live] = t;
          new_cum[live] = cand_s[r];
        }
        ++live;
      }
    }
    __syncwarp();
    int d = 0;
    if (c + 1 >= limit) {
      for (int w = 0; w < live; ++w) insert((float)((double)new_cum[w] / len_pow[0]), MAX_W + w, (int)c + 1);
      d = c + 1 >= max_seq_len ? 3 : 2;
    } else if (live == 0) {
      d = 1;
    } else if (fins >= W) {
      uint32_t low;
      lowest(low);
      float best = lane < live ? new_cum[lane] : neg_inf();
      if (lane + 32 < live) best = fmaxf(best, new_cum[lane + 32]);
      best = warp_max(best);
      const double ahead = fmax((double)best / len_pow[1], (double)best / len_pow[2]);
      if (early || (double)key_value(low) >= ahead) d = 1;
    }
    if (lane < W) {
      st.fin_score[g * W + lane] = fin0;
      st.fin_len[g * W + lane] = len0;
    }
    if (lane + 32 < W) {
      st.fin_score[g * W + lane + 32] = fin1;
      st.fin_len[g * W + lane + 32] = len1;
    }
    if (lane == 0) {
      live_n = live;
      st.fin_count[g] = fins;
      st.count[g] = (int32_t)(c + 1);
      st.done[g] = (uint8_t)d;
    }
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
  if (tid < W) {
    if (tid < live) {
      hist[tid * st.cap + c] = new_tok[tid];
      st.last[g * W + tid] = new_tok[tid];
    }
    st.cum[g * W + tid] = new_cum[tid];
    st.parent[g * W + tid] = new_par[tid];
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
// Bound by HBM: 32 caches of 64 beams x 4 heads x 1100 x 128 bf16 take 539 us
// out of place (the rows written and the distinct parents read: 7.1 TB/s), two
// of them 36 us.
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
