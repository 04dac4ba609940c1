// The vocabulary projection's weight in 4 bits with group scales (pesti_q4_*), and logits from it.
//
//   s = bf16(-m / 8), m the group's largest value by magnitude (the first of equal ones)
//   q = clamp(rint(w / s), -8, 7),  y = x (q s)^T
//
// Layout.  A row is padded to blocks of 128 columns of 64 bytes; word 4 t + j of a block (t, j = 0..3) holds columns
// 32 j + 8 t to + 7, eight nibbles q + 8 from its low end.  So 16 bytes at word 4 t are what lane t of a quad of an
// m16n8k16 product needs for four steps of 32 columns, none of which crosses a group.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "pesti_common.cuh"
#include "pesti_umma.cuh"

namespace pesti_q4 {

constexpr int BLOCK = 128;  // columns
constexpr int BLOCK_BYTES = BLOCK / 2;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __half2float(v);
  else
    return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(v);
  else
    return __float2bfloat16_rn(v);
}

// The word of columns 8 i to 8 i + 7 of a block: i = 4 j + t is at 4 t + j.
__device__ __forceinline__ int word_of(int i) { return (i & 3) * 4 + (i >> 2); }

template <typename T>
struct Held {
  const T* w;
  long long ld;
  uint32_t* q;
  __nv_bfloat16* scale;
  int D, blocks, runs;  // blocks of a row, and runs of PER blocks that half a warp takes
  long long total;      // runs in all
  int vec;              // whole vectors of 8 columns can be read or written
};

// The row and the first block of a team of LANES lanes.
template <typename T, int PER, int LANES>
__device__ __forceinline__ bool place_of(const Held<T>& a, long long& row, int& block) {
  const long long run = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  row = a.total >> 32 ? run / a.runs : (uint32_t)run / (uint32_t)a.runs;
  block = (int)(run - row * a.runs) * PER;
  return run < a.total;
}

// Quotients w / s as codes q + 8, rounded to whole numbers, halves to even, exactly.  t = 384 + w / s to 2^-15 (the
// spacing of numbers about 384), off by at most 2^-20 before that, since |w / s| < 8.1; adding 1.5 * 2^23 rounds it to
// whole numbers, which the sum's last bits hold.
//  16-bit w: of 11 bits, and s of 8, so that a quotient that is no half is at least 2^-13 from one: rounding to 2^-15
//  brings back the halves and moves nothing across one.
//  f32 w: quotients within 2^-14 of a half are looked at again, with the exact remainder (w has 24 bits, q s at most
//  12, and a quotient off by less than one leaves an f32).
constexpr float WHOLE = 12582912.0f;  // 1.5 * 2^23

__device__ __forceinline__ uint32_t codes_of(const float (&v)[8], float s, bool check) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  uint32_t word = 0;
  float far = 0.0f;
  // (the eight sums' upper bits, 0x4b400000, add up to this constant)
  constexpr uint32_t UPPER = 0x4b400000u + (0x4b400000u << 4) + (0x4b400000u << 8);
#pragma unroll
  for (int j = 7; j >= 0; --j) {
    const float t = fminf(fmaf(v[j], inv, 384.0f), 391.0f), c = t + (WHOLE + 8.0f - 384.0f);
    word = (word << 4) + fbits(c);
    if (check) far = fmaxf(far, fabsf((c - (WHOLE + 8.0f - 384.0f)) - t));
  }
  word -= UPPER;
  if (check && far >= 0.5f - 0x1p-14f) {
    word = 0;
#pragma unroll 1
    for (int j = 7; j >= 0; --j) {
      float w = v[0];
#pragma unroll
      for (int i = 1; i < 8; ++i)
        if (i == j) w = v[i];
      float q = rintf(w * inv);
      const float r = fmaf(-q, s, w), r2 = 2.0f * fabsf(r), a = fabsf(s);
      if (r2 > a || (r2 == a && ((int)q & 1))) q += (r > 0.0f) == (s > 0.0f) ? 1.0f : -1.0f;
      word = (word << 4) + (uint32_t)((int)fminf(q, 7.0f) + 8);
    }
  }
  return word;
}

// The larger of two pairs, NaN where one of them is.
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, bool f16) {
  uint32_t r;
  if (f16)
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sixteen columns of a lane as they were read: f32, or pairs of 16 bits.
template <typename T>
struct Sixteen {
  static constexpr int WORDS = 4 * sizeof(T);
  uint32_t v[WORDS];

  __device__ __forceinline__ void load(const T* row, int at, int D, bool vec) {
    if (vec && at + 16 <= D) {
#pragma unroll
      for (int i = 0; i < WORDS; i += 8)
        asm volatile("ld.global.cs.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]),
                       "=r"(v[i + 6]), "=r"(v[i + 7])
                     : "l"((const uint32_t*)(row + at) + i));
    } else {
      T* p = (T*)v;
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = at + i < D ? row[at + i] : from_f32<T>(0.0f);
    }
  }

  __device__ __forceinline__ float at(int i) const { return to_f32(((const T*)v)[i]); }

  // The largest value and the largest negated one of GROUP / 16 lanes' columns.
  template <int GROUP>
  __device__ __forceinline__ void ends(float& hi, float& neg) const {
    if constexpr (sizeof(T) == 4) {
      hi = bitsf(v[0]);
      neg = -hi;
#pragma unroll
      for (int i = 1; i < WORDS; ++i) {
        hi = max_nan(hi, bitsf(v[i]));
        neg = max_nan(neg, -bitsf(v[i]));
      }
#pragma unroll
      for (int o = 1; o < GROUP / 16; o <<= 1) {
        hi = max_nan(hi, __shfl_xor_sync(PESTI_FULL_MASK, hi, o));
        neg = max_nan(neg, __shfl_xor_sync(PESTI_FULL_MASK, neg, o));
      }
    } else {
      constexpr bool F16 = std::is_same<T, __half>::value;
      constexpr uint32_t SIGNS = 0x80008000u;
      uint32_t a = v[0], b = v[0] ^ SIGNS;
#pragma unroll
      for (int i = 1; i < WORDS; ++i) {
        a = max2_nan(a, v[i], F16);
        b = max2_nan(b, v[i] ^ SIGNS, F16);
      }
      uint32_t both = max2_nan(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), F16);  // (value, negated)
#pragma unroll
      for (int o = 1; o < GROUP / 16; o <<= 1) both = max2_nan(both, __shfl_xor_sync(PESTI_FULL_MASK, both, o), F16);
      const T* p = (const T*)&both;
      hi = to_f32(p[0]);
      neg = to_f32(p[1]);
    }
  }
};

// Eight lanes a block of 128 columns, 16 columns and two words each; PER blocks at once for the loads in flight.  The
// 16-bit forms are bound by instructions (10 a column; 8 columns a lane took 19 more a column): 128256 x 4096 bf16, see
// q4_dequantize_kernel for the way back.
template <typename T, int GROUP, int PER>
__global__ void __launch_bounds__(256) q4_quantize_kernel(const Held<T> a) {
  const int i = threadIdx.x & 7, lane = threadIdx.x & 31;
  long long row;
  int b0;
  const bool there = place_of<T, PER, 8>(a, row, b0);
  const int n = there ? min(PER, a.blocks - b0) : 0;
  Sixteen<T> in[PER];
  const T* from = a.w + row * a.ld;
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (u < n) in[u].load(from, (b0 + u) * BLOCK + 16 * i, a.D, a.vec);
  const long long b = row * a.blocks + b0;
  uint32_t* to = a.q + b * (BLOCK / 8) + word_of(2 * i);  // (the other word is 4 behind it)
  __nv_bfloat16* scale = a.scale + b * (BLOCK / GROUP) + i / (GROUP / 16);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    float hi, neg;
    in[u].template ends<GROUP>(hi, neg);
    float m = hi > neg ? hi : -neg;
    if (__any_sync(PESTI_FULL_MASK, hi == neg)) {  // both signs: the one that comes first
      int first = 32 * 32;
#pragma unroll
      for (int j = 15; j >= 0; --j)
        if (fabsf(in[u].at(j)) == hi) first = 2 * (16 * lane + j) + (in[u].at(j) < 0.0f ? 1 : 0);
#pragma unroll
      for (int o = 1; o < GROUP / 16; o <<= 1) first = min(first, __shfl_xor_sync(PESTI_FULL_MASK, first, o));
      if (hi == neg) m = first & 1 ? -hi : hi;
    }
    if (u >= n) continue;
    __nv_bfloat16 held = __float2bfloat16_rn(m * -0.125f);
    float s = __bfloat162float(held);
    uint32_t word[2] = {0x88888888u, 0x88888888u};
    if (!isfinite(m)) {
      held = __float2bfloat16_rn(NAN);
    } else if (s != 0.0f) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8], t = s;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = in[u].at(8 * h + j);
        if (fabsf(s) < 0x1p-100f) {  // so that 1 / s is finite, and quotients by subnormal scales at most 8
          t = s * 0x1p64f;
          const float most = 8.0f * fabsf(t);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = fminf(most, fmaxf(-most, v[j] * 0x1p64f));
        }
        word[h] = codes_of(v, t, sizeof(T) == 4);
      }
    }
    to[u * (BLOCK / 8)] = word[0];
    to[u * (BLOCK / 8) + 4] = word[1];
    if (i % (GROUP / 16) == 0) scale[u * (BLOCK / GROUP)] = held;
  }
}

// Two lanes of a team of sixteen hold neighbouring words; f32 rows are written 32 bytes a lane, 16-bit ones 16.
template <typename T, int GROUP, int PER>
__global__ void __launch_bounds__(256) q4_dequantize_kernel(const Held<T> a) {
  const int i = threadIdx.x & 15;
  long long row;
  int b0;
  if (!place_of<T, PER, 16>(a, row, b0)) return;
  const int n = min(PER, a.blocks - b0);
  const long long b = row * a.blocks + b0;
  const uint32_t* from = a.q + b * (BLOCK / 8) + word_of(i);
  const __nv_bfloat16* scale = a.scale + b * (BLOCK / GROUP) + i / (GROUP / 8);
  uint32_t w[PER];
  float s[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (u < n) {
      w[u] = __ldcs(from + u * (BLOCK / 8));
      s[u] = __bfloat162float(scale[u * (BLOCK / GROUP)]);
    }
  }
  T* to = const_cast<T*>(a.w) + row * a.ld;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (u >= n) continue;
    const int at = (b0 + u) * BLOCK + 8 * i;
    uint32_t raw[2 * sizeof(T)];
    T* v = (T*)raw;
#pragma unroll
    for (int j = 0; j < 8; ++j)  // 2^23 + 8 + q from the nibble, less 2^23 + 8
      v[j] = from_f32<T>((bitsf(((w[u] >> (4 * j)) & 15u) | 0x4b000000u) - 8388616.0f) * s[u]);
    if (a.vec && at + 8 <= a.D) {
      if constexpr (sizeof(T) == 4)
        asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + at), "r"(raw[0]),
                     "r"(raw[1]), "r"(raw[2]), "r"(raw[3]), "r"(raw[4]), "r"(raw[5]), "r"(raw[6]), "r"(raw[7])
                     : "memory");
      else
        __stcs((uint4*)(to + at), make_uint4(raw[0], raw[1], raw[2], raw[3]));
    } else {
      for (int j = 0; j < 8 && at + j < a.D; ++j) to[at + j] = v[j];
    }
  }
}

// --- logits

struct LogitArgs {
  const void* x;
  long long x_ld;
  int rows, D;  // of x; at most 64 rows
  const uint4* q;
  const __nv_bfloat16* scale;
  int V, blocks, tiles;  // 32 rows of the weight a tile
  uint4* frags;          // [blocks][4][pieces][8 NT][4], where x does not fit shared memory whole
  void* y;
  long long y_ld;
  int out;               // 0 f32, 1 bf16, 2 f16
  int warps, k_warps;    // warps that multiply, and how many of them share a tile's K
  int stage_blocks, stages;
};

// The bf16 or f16 bits of piece `p` of an x: f32 is cut into three bf16 whose sum it is, exactly.
template <typename T>
__device__ __forceinline__ uint32_t piece_of(T x, int p) {
  if constexpr (sizeof(T) == 2) {
    return *(const uint16_t*)&x;
  } else {
    float rest = x;
    uint32_t bits = fbits(rest);
    for (int i = 0; i < p; ++i) {
      const bool whole = (bits & 0x7f800000u) == 0x7f800000u;  // inf and NaN are in the first piece
      rest = whole ? 0.0f : rest - bitsf(bits & 0xffff0000u);
      bits = fbits(rest);
    }
    return bits >> 16 | (is_nan(rest) ? 0x40u : 0u);
  }
}

// Four pairs of x for lane t of a quad, word j of block b: columns 32 j + 8 t + (i, i + 4), as a word of weights unpacks.
template <typename T>
__device__ __forceinline__ uint4 fragment_of(const T* row, int b, int j, int t, int piece, int D) {
  const int at = b * BLOCK + 32 * j + 8 * t;
  uint32_t v[8], f[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = at + i < D ? piece_of(row[at + i], piece) : 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = v[i] | v[i + 4] << 16;
  return make_uint4(f[0], f[1], f[2], f[3]);
}

template <typename T>
__global__ void __launch_bounds__(256) q4_fragments_kernel(const LogitArgs a, int columns) {
  pesti_umma::depend_wait();
  pesti_umma::depend_launch();
  constexpr int P = sizeof(T) == 4 ? 3 : 1;
  const int per_block = 16 * P * columns;
  for (int e = threadIdx.x; e < per_block; e += 256) {
    const int t = e & 3, c = (e >> 2) % columns, jp = (e >> 2) / columns, p = jp % P, j = jp / P;
    uint4 f = make_uint4(0, 0, 0, 0);
    if (c < a.rows) f = fragment_of((const T*)a.x + c * a.x_ld, blockIdx.x, j, t, p, a.D);
    a.frags[(long long)blockIdx.x * per_block + e] = f;
  }
}

// Nibbles i and i + 4 of a word as two 16-bit floats q: the nibble becomes the mantissa's low end of 128 (bf16) or
// 1024 (f16), and 8 more than that is taken off, exactly.
template <bool F16>
__device__ __forceinline__ uint32_t unpack(uint32_t word, int i) {
  uint32_t v;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(v) : "r"(word >> (4 * i)), "r"(F16 ? 0x64006400u : 0x43004300u));
  if constexpr (F16) {
    const __half2 r = __hsub2(*(__half2*)&v, __half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408)));
    return *(const uint32_t*)&r;
  } else {
    const __nv_bfloat162 r =
        __hsub2(*(__nv_bfloat162*)&v, __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)));
    return *(const uint32_t*)&r;
  }
}

template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int ROWS = 32;  // of the weight, per warp and tile

__host__ __device__ constexpr int most_warps(int nt) { return nt <= 2 ? 15 : nt == 4 ? 11 : 7; }

// A lane's weights of one block: 16 bytes of four rows (8 apart), and their groups' scales.
template <int GROUP>
struct Weights {
  uint4 w[4];
  uint2 s[4];  // up to four bf16

  __device__ __forceinline__ void load(const uint4* const (&q)[4], const __nv_bfloat16* const (&sc)[4], int b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = __ldcs(q[i] + b * (BLOCK_BYTES / 16));
      const __nv_bfloat16* p = sc[i] + b * (BLOCK / GROUP);
      if constexpr (GROUP == 32)
        s[i] = __ldg((const uint2*)p);
      else if constexpr (GROUP == 64)
        s[i].x = __ldg((const uint32_t*)p);
      else
        s[i].x = __ldg((const uint16_t*)p);
    }
  }

  __device__ __forceinline__ float scale(int i, int g) const {
    const uint32_t v = g < 2 ? s[i].x : s[i].y;
    return bitsf(g & 1 ? v & 0xffff0000u : v << 16);
  }
};

__device__ __forceinline__ void multipliers_sync(int threads) {
  asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}

// A warp multiplies 32 rows of the weight by all columns of x over its share of K (every k_warps-th block), and goes on
// to its next tile; the k_warps warps of a tile join their sums in shared memory, in their order.  Blocks of weights are
// loaded two ahead of their products.  Columns past x's last row hold zeros.
// RING: x passes through shared memory in stages, copied by a warp of its own, again for every round of tiles.
// Otherwise x is laid out there once, by all warps, while the first weights are on their way.
template <typename T, int GROUP, int NT, bool RING>
__global__ void __launch_bounds__((most_warps(NT) + 1) * 32) q4_logits_kernel(const LogitArgs a) {
  using namespace pesti_umma;
  constexpr bool F16 = std::is_same<T, __half>::value;
  constexpr int P = sizeof(T) == 4 ? 3 : 1, COLUMNS = 8 * NT;
  extern __shared__ uint4 xs[];
  __shared__ uint64_t bars[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kw = a.k_warps, slots = a.warps / kw, part = warp % kw, slot = warp / kw;
  const int columns = RING ? COLUMNS : a.rows;  // in shared memory
  const int per_block = 16 * P * columns;       // 16-byte fragments of a block of x
  const int rounds = (a.tiles + gridDim.x * slots - 1) / (gridDim.x * slots);
  const uint32_t full = smem_addr(bars), empty = full + 64;
  float* sums = (float*)(xs + (long long)(RING ? a.stages * a.stage_blocks : a.blocks) * per_block);

  if (RING && threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      bar_init(full + 8 * s, 1);
      bar_init(empty + 8 * s, a.warps);
    }
    bar_init_fence();
  }
  if (RING) __syncthreads();
  depend_launch();

  if (RING && warp == a.warps) {  // copies x
    if (lane == 0) {
      depend_wait();
      int s = 0, ph = 0;
      bool ok = true;
      for (int r = 0; r < rounds && ok; ++r) {
        for (int b = 0; b < a.blocks; b += a.stage_blocks) {
          ok = bar_wait(empty + 8 * s, ph ^ 1);
          if (!ok) break;
          const uint32_t bytes = min(a.stage_blocks, a.blocks - b) * per_block * 16;
          bar_expect(full + 8 * s, bytes);
          bulk_load(smem_addr(xs + (long long)s * a.stage_blocks * per_block), a.frags + (long long)b * per_block,
                    full + 8 * s, bytes);
          if (++s == a.stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
    return;
  }

  // the next block to load: its tile's round, and its place
  const uint4* q[4];
  const __nv_bfloat16* sc[4];
  auto rows_of = [&](int round) {
    const int tile = min(((int)blockIdx.x + round * (int)gridDim.x) * slots + slot, a.tiles - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = min(tile * ROWS + g + 8 * i, a.V - 1);
      q[i] = a.q + (row * a.blocks) * (BLOCK_BYTES / 16) + t;
      sc[i] = a.scale + (row * a.blocks) * (BLOCK / GROUP);
    }
  };
  int load_round = 0, load_b = part;
  rows_of(0);
  Weights<GROUP> held[2];
  auto load = [&](Weights<GROUP>& w) {
    if (load_round >= rounds) return;
    w.load(q, sc, load_b);
    load_b += kw;
    if (load_b >= a.blocks) {
      load_b = part;
      if (++load_round < rounds) rows_of(load_round);
    }
  };
  load(held[0]);
  load(held[1]);

  if (!RING) {
    depend_wait();
    for (int e = threadIdx.x; e < a.blocks * per_block; e += a.warps * 32) {
      const int tt = e & 3, rest = e >> 2, c = rest % columns, bjp = rest / columns, p = bjp % P, bj = bjp / P;
      xs[e] = fragment_of((const T*)a.x + c * a.x_ld, bj >> 2, bj & 3, tt, p, a.D);
    }
    __syncthreads();
  }

  float acc[2][NT][4];
  int s = 0, ph = 0, which = 0;
  bool ok = true;

  // the products of block b with the fragments at `x`
  auto multiply = [&](Weights<GROUP>& w, const uint4* x) {
#pragma unroll
    for (int gr = 0; gr < BLOCK / GROUP; ++gr) {
      float part_acc[2][NT][4] = {};
#pragma unroll
      for (int jj = 0; jj < GROUP / 32; ++jj) {
        const int j = gr * (GROUP / 32) + jj;
        uint32_t fa[2][2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w0 = ((const uint32_t*)&w.w[2 * m])[j], w1 = ((const uint32_t*)&w.w[2 * m + 1])[j];
            fa[m][h][0] = unpack<F16>(w0, 2 * h);
            fa[m][h][1] = unpack<F16>(w1, 2 * h);
            fa[m][h][2] = unpack<F16>(w0, 2 * h + 1);
            fa[m][h][3] = unpack<F16>(w1, 2 * h + 1);
          }
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint4 f = make_uint4(0, 0, 0, 0);
            const int c = n * 8 + g;
            if (RING || c < columns) f = x[((j * P + p) * columns + c) * 4 + t];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              mma<F16>(part_acc[m][n], fa[m][0], f.x, f.y);
              mma<F16>(part_acc[m][n], fa[m][1], f.z, f.w);
            }
          }
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float s0 = w.scale(2 * m, gr), s1 = w.scale(2 * m + 1, gr);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[m][n][0] = fmaf(s0, part_acc[m][n][0], acc[m][n][0]);
          acc[m][n][1] = fmaf(s0, part_acc[m][n][1], acc[m][n][1]);
          acc[m][n][2] = fmaf(s1, part_acc[m][n][2], acc[m][n][2]);
          acc[m][n][3] = fmaf(s1, part_acc[m][n][3], acc[m][n][3]);
        }
      }
    }
    load(w);
  };

  for (int r = 0; r < rounds; ++r) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.0f;
    if (RING) {
      for (int b0 = 0; b0 < a.blocks; b0 += a.stage_blocks) {
        if (ok) ok = bar_wait(full + 8 * s, ph);
        const uint4* x = xs + (long long)s * a.stage_blocks * per_block;
        const int b1 = min(b0 + a.stage_blocks, a.blocks);
        for (int b = b0 + part; b < b1; b += kw) {
          if (which)
            multiply(held[1], x + (b - b0) * per_block);
          else
            multiply(held[0], x + (b - b0) * per_block);
          which ^= 1;
        }
        __syncwarp();
        if (lane == 0) bar_arrive_cluster(empty + 8 * s);
        if (++s == a.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    } else {
      for (int b = part; b < a.blocks; b += kw) {
        if (which)
          multiply(held[1], xs + b * per_block);
        else
          multiply(held[0], xs + b * per_block);
        which ^= 1;
      }
    }
    const int tile = ((int)blockIdx.x + r * (int)gridDim.x) * slots + slot;
    if (kw > 1) {
      // [slot][part - 1][values][lane]
      float* to = sums + ((long long)slot * (kw - 1) + (part - 1)) * (8 * NT) * 32 + lane;
      if (part) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) to[((m * NT + n) * 4 + e) * 32] = acc[m][n][e];
      }
      multipliers_sync(a.warps * 32);
      if (!part) {
        for (int k = 1; k < kw; ++k) {
          const float* from = sums + ((long long)slot * (kw - 1) + (k - 1)) * (8 * NT) * 32 + lane;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[m][n][e] += from[((m * NT + n) * 4 + e) * 32];
        }
      }
      multipliers_sync(a.warps * 32);
    }
    if (part == 0 && tile < a.tiles) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = n * 8 + 2 * t + (e & 1), v = tile * ROWS + 16 * m + 8 * (e >> 1) + g;
            if (c >= a.rows || v >= a.V) continue;
            const float y = ok ? acc[m][n][e] : NAN;  // NaN: a wait gave up
            const long long at = c * a.y_ld + v;
            if (a.out == 0)
              ((float*)a.y)[at] = y;
            else if (a.out == 1)
              ((__nv_bfloat16*)a.y)[at] = __float2bfloat16_rn(y);
            else
              ((__half*)a.y)[at] = __float2half_rn(y);
          }
    }
  }
}

}  // namespace pesti_q4
