// The vocabulary projection's weight in 4 bits with group scales (pesti_q4_*), and logits from it.
//
//   s = bf16(-m / 8), m the group's largest value by magnitude (the first of equal ones)
//   q = clamp(rint(w / s), -8, 7),  y = x (q s)^T
//
// Layout.  Tiles of 64 rows and 128 columns of 4 KB, [ceil(V / 64)][ceil(D / 128)][64 rows][64 bytes].  A row's 16-byte
// chunk t is at place t ^ (row / 2 % 4), and its word j holds columns 32 j + 8 t to + 7: eight nibbles q + 8 from its low
// end.  So a chunk is what lane t of a quad of an m16n8k16 product needs for four steps of 32 columns, none of which
// crosses a group; a tile is one copy; and its rows' chunks are read from shared memory without bank conflicts, by quads
// or by threads that take a row each.  Scales: [ceil(V / 64)][ceil(D / 128)][64 rows][128 / group].
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

constexpr int ROWS = 64;                          // of a tile
constexpr int TILE_WORDS = ROWS * BLOCK_BYTES / 4;

// Where chunk t of a row is among the row's four.
__host__ __device__ __forceinline__ int chunk_at(int row, int t) { return t ^ (row >> 1 & 3); }

// The tile of a row's block, and in it the word of its columns 8 i to 8 i + 7, i = 4 j + t.
__device__ __forceinline__ long long tile_of(long long row, int blocks, int block) { return (row >> 6) * blocks + block; }
__device__ __forceinline__ int word_of(int row, int i) {
  return (row & 63) * (BLOCK_BYTES / 4) + chunk_at(row, i & 3) * 4 + (i >> 2);
}

template <typename T>
struct Held {
  const T* w;
  long long ld;
  uint32_t* q;
  __nv_bfloat16* scale;
  int D, blocks, runs;  // blocks of a row, and runs of PER blocks that its team takes
  int V;
  long long total;      // runs of all rows, or of all sixteens of rows
  int vec;              // whole vectors of 8 columns can be read or written
};

// What a team of lanes takes of `total` runs: which of the first index's, and which of `runs` behind it.
__device__ __forceinline__ bool place_of(long long team, long long total, int runs, long long& first, int& run) {
  first = total >> 32 ? team / runs : (uint32_t)team / (uint32_t)runs;
  run = (int)(team - first * runs);
  return team < total;
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

// Eight lanes a block of 128 columns, 16 columns and two words each; PER blocks at once for the loads in flight.  f32 is
// bound by HBM, 16 bits by instructions: 128256 x 4096 in 385 us f32 (6.2 TB/s), 235 us bf16 (5.6 TB/s, 13 instructions
// a column; with 8 columns a lane 20, and 322 us).
template <typename T, int GROUP, int PER>
__global__ void __launch_bounds__(256) q4_quantize_kernel(const Held<T> a) {
  const int i = threadIdx.x & 7, lane = threadIdx.x & 31;
  // teams along a row, which reads best
  long long row;
  int b0;
  const bool there = place_of((long long)blockIdx.x * 32 + (threadIdx.x >> 3), a.total, a.runs, row, b0);
  b0 *= PER;
  const int n = there ? min(PER, a.blocks - b0) : 0;
  Sixteen<T> in[PER];
  const T* from = a.w + row * a.ld;
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (u < n && row < a.V) in[u].load(from, (b0 + u) * BLOCK + 16 * i, a.D, a.vec);
  const long long b = tile_of(row, a.blocks, b0);
  const bool real = row < a.V;  // (rows to a whole tile are held as zeros)
  uint32_t* to = a.q + b * TILE_WORDS;
  const int word0 = word_of(row, 2 * i), word1 = word_of(row, 2 * i + 1);
  __nv_bfloat16* scale = a.scale + (b * ROWS + (row & 63)) * (BLOCK / GROUP) + i / (GROUP / 16);
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
    to[u * TILE_WORDS + word0] = real ? word[0] : 0x88888888u;
    to[u * TILE_WORDS + word1] = real ? word[1] : 0x88888888u;
    if (i % (GROUP / 16) == 0) scale[u * ROWS * (BLOCK / GROUP)] = real ? held : __nv_bfloat16(0.0f);
  }
}

// f32 rows are written 32 bytes a lane (128256 x 4096 in 370 us; by 16 bytes 475), 16-bit ones 16 (bf16: 230 us, 5.7 TB/s).
template <typename T, int GROUP, int PER>
__global__ void __launch_bounds__(256) q4_dequantize_kernel(const Held<T> a) {
  const int i = threadIdx.x & 15;
  // sixteen teams for sixteen rows of a tile, whose bytes are next to one another
  long long row;
  int b0;
  if (!place_of(blockIdx.x, a.total, a.runs, row, b0)) return;
  row = row * 16 + (threadIdx.x >> 4);
  b0 *= PER;
  if (row >= a.V) return;
  const int n = min(PER, a.blocks - b0);
  const long long b = tile_of(row, a.blocks, b0);
  const uint32_t* from = a.q + b * TILE_WORDS + word_of(row, i);
  const __nv_bfloat16* scale = a.scale + (b * ROWS + (row & 63)) * (BLOCK / GROUP) + i / (GROUP / 8);
  uint32_t w[PER];
  float s[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (u < n) {
      w[u] = __ldcs(from + u * TILE_WORDS);
      s[u] = __bfloat162float(scale[u * ROWS * (BLOCK / GROUP)]);
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
  int x_vec;    // whole vectors of 8 columns can be read
  const uint4* q;
  const __nv_bfloat16* scale;
  int V, blocks, stacks;  // tiles of 64 rows, or pairs of them
  uint4* operand;        // x for the tensor cores (q4_operand_kernel)
  int stages;            // blocks in shared memory at once
  void* y;
  long long y_ld;
  int out;               // 0 f32, 1 bf16, 2 f16
  int k_warps;           // warps that share a tile's K
  int give_up;           // for tests: which of a slot's rounds is taken for one whose wait gave up (-1: none)
};

__device__ __forceinline__ void store_logit(const LogitArgs& a, int row, int v, float y) {
  const long long at = row * a.y_ld + v;
  if (a.out == 0)
    ((float*)a.y)[at] = y;
  else if (a.out == 1)
    ((__nv_bfloat16*)a.y)[at] = __float2bfloat16_rn(y);
  else
    ((__half*)a.y)[at] = __float2half_rn(y);
}

// f32 x enters the products as a sum of two f16, times a power of two of its row that brings the row's largest finite
// value to 2^14 or more: off by at most 2^-24 of itself or 2^-39 of that value, which is below what an f32 sum of the
// products loses.  (Three bf16, exact without a power of two, cost a product more, 97 us instead of 77 for a row of
// 128256 x 4096.)  16-bit x enters them as it is, or (IN_F16) bf16 as f16 times such a power: exactly, down to 2^-39 of
// the row's largest value.
template <typename T>
constexpr int pieces = sizeof(T) == 4 ? 2 : 1;
template <typename T>
constexpr bool in_bf16 = std::is_same<T, __nv_bfloat16>::value;
template <typename T, bool IN_F16>
constexpr bool scaled = sizeof(T) == 4 || (IN_F16 && in_bf16<T>);

// Eight columns of a row of x.
template <typename T>
struct EightX {
  uint32_t raw[2 * sizeof(T)];

  __device__ __forceinline__ void load(const T* row, int at, int D, bool vec) {
    if (vec && at + 8 <= D) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) *((uint4*)raw + i) = *((const uint4*)(row + at) + i);
    } else {
      T* v = (T*)raw;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = at + i < D ? row[at + i] : from_f32<T>(0.0f);
    }
  }

  __device__ __forceinline__ float at(int i) const { return to_f32(((const T*)raw)[i]); }

  // The largest finite magnitude.
  __device__ __forceinline__ float most() const {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, isfinite(at(i)) ? fabsf(at(i)) : 0.0f);
    return m;
  }

  // The pairs (i, i + 4) that a word of weights unpacks to (scaled: times up.x * up.y).
  template <bool IN_F16>
  __device__ __forceinline__ void fragments(float2 up, uint4 (&f)[pieces<T>]) const {
    if constexpr (!scaled<T, IN_F16>) {
      f[0] = make_uint4(__byte_perm(raw[0], raw[2], 0x5410), __byte_perm(raw[0], raw[2], 0x7632),
                        __byte_perm(raw[1], raw[3], 0x5410), __byte_perm(raw[1], raw[3], 0x7632));
    } else {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = at(i) * up.x * up.y;
#pragma unroll
      for (int p = 0; p < pieces<T>; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half lo = __float2half_rn(v[i]), hi = __float2half_rn(v[i + 4]);
          w[i] = (uint32_t)__half_as_ushort(lo) | (uint32_t)__half_as_ushort(hi) << 16;
          // an infinity or a NaN is in the first of two
          v[i] = isfinite(v[i]) ? v[i] - __half2float(lo) : 0.0f;
          v[i + 4] = isfinite(v[i + 4]) ? v[i + 4] - __half2float(hi) : 0.0f;
        }
        f[p] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
};

// The row's power of two as a product of two f32, and its inverse.
__device__ __forceinline__ float2 row_scale(float most, bool inverse) {
  if (most == 0.0f) return make_float2(1.0f, 1.0f);
  const int e = inverse ? ilogbf(most) - 14 : 14 - ilogbf(most), a = e / 2;
  return make_float2(bitsf((uint32_t)(a + 127) << 23), bitsf((uint32_t)(e - a + 127) << 23));
}

// Nibbles i and i + 4 of a word as two 16-bit floats q: a nibble becomes the mantissa's low end of 128 (bf16) or 1024
// (f16), and 8 more than that is taken off, exactly.  In f16 16 times a nibble does as well, which takes no shift.
__device__ __forceinline__ uint32_t masked(uint32_t word, uint32_t mask, uint32_t upper) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(word), "r"(mask), "r"(upper));
  return v;
}
template <bool BF16>
__device__ __forceinline__ void unpack(uint32_t word, uint32_t (&q)[4]) {
  if constexpr (BF16) {
    const __nv_bfloat162 low = __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));  // 136
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = masked(word >> (4 * i), 0x000f000fu, 0x43004300u);
      const __nv_bfloat162 r = __hsub2(*(const __nv_bfloat162*)&v, low);
      q[i] = *(const uint32_t*)&r;
    }
  } else {
    const __half2 low = __half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));   // 1032
    const __half2 part = __half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));  // 1 / 16
    const __half2 high = __half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));  // -72
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = masked(i < 2 ? word : word >> 8, i & 1 ? 0x00f000f0u : 0x000f000fu, 0x64006400u);
      const __half2 x = *(const __half2*)&v, r = i & 1 ? __hfma2(x, part, high) : __hsub2(x, low);
      q[i] = *(const uint32_t*)&r;
    }
  }
}

// c (+)= A B over 16 of K.
template <bool BF16, bool ADD>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  const float z0 = ADD ? c[0] : 0.0f, z1 = ADD ? c[1] : 0.0f, z2 = ADD ? c[2] : 0.0f, z3 = ADD ? c[3] : 0.0f;
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
}

// A lane's weights of 16 rows of a tile: 16 bytes of two rows (8 apart), and their groups' scales.
template <int GROUP>
struct Weights {
  uint4 w[2];
  uint2 s[2];  // up to four bf16

  __device__ __forceinline__ void load(const uint4* q, const __nv_bfloat16* sc) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = __ldcs(q + i * 8 * (BLOCK_BYTES / 16));
      const __nv_bfloat16* p = sc + i * 8 * (BLOCK / GROUP);
      if constexpr (GROUP == 32)
        s[i] = __ldcs((const uint2*)p);
      else if constexpr (GROUP == 64)
        s[i].x = __ldcs((const uint32_t*)p);
      else
        s[i].x = __ldcs((const uint16_t*)p);
    }
  }

  __device__ __forceinline__ float scale(int i, int g) const {
    const uint32_t v = g < 2 ? s[i].x : s[i].y;
    return bitsf(g & 1 ? v & 0xffff0000u : v << 16);
  }
};

// Warps that multiply: their registers hold a tile's sums, the next weights and the fragments of a block of x.
constexpr int FEW_WARPS = 16;

// Barriers 1 to 7 and 8 to 14 of a block, one for each slot.
constexpr int MOST_SLOTS = 7;
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void named_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Up to 8 rows of x: a warp multiplies a tile of 64 rows of the weight by all of them over its share of K (every
// k_warps-th block), and goes on to its next tile; the k_warps warps of a tile join their sums in shared memory, in
// their order.  x is laid out in shared memory once, while the first weights are on their way; a tile's weights are
// loaded a block ahead, and on their way to L2 another block ahead.  A row of 128256 x 4096, g 64: 60 us in bf16, 56 in
// f16, 74 in f32 (4.7 to 3.8 TB/s), bound by the integer pipe that unpacks; with tiles of 16 rows, 1 KB at a time, 64.
// Of 32000 x 2048, g 32: 11.5 us, without the prefetch 13.9.  Copies into four stages of shared memory: 59 and 11.5, but
// 8 rows of 64000 x 8192, which leave them no room, 80 instead of 68.
template <typename T, int GROUP>
__global__ void __launch_bounds__(FEW_WARPS * 32, 1) q4_logits_kernel(const LogitArgs a) {
  constexpr bool BF16 = in_bf16<T>;
  constexpr int P = pieces<T>, WARPS = FEW_WARPS;
  extern __shared__ uint4 xs[];
  __shared__ float most[8];  // of each row of x
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kw = a.k_warps, slots = WARPS / kw, part = warp % kw, slot = warp / kw;
  const int columns = a.rows, per_block = 16 * P * columns;  // 16-byte fragments of a block of x
  const int rounds = (a.stacks + gridDim.x * slots - 1) / (gridDim.x * slots);
  float* sums = (float*)(xs + a.blocks * per_block + 1);
  pesti_umma::depend_wait();
  pesti_umma::depend_launch();

  // the block to load next, of the tile of `load_round`
  const uint4* q;
  const __nv_bfloat16* sc;
  int load_round = 0, load_b = part;
  Weights<GROUP> held[4];
  auto stack_of = [&](int round) { return (round * (int)gridDim.x + (int)blockIdx.x) * slots + slot; };
  auto begin = [&]() {
    const long long tile = (long long)min(stack_of(load_round), a.stacks - 1) * a.blocks + part;
    q = a.q + tile * (TILE_WORDS / 4) + g * 4 + chunk_at(g, t);
    sc = a.scale + (tile * ROWS + g) * (BLOCK / GROUP);
  };
  auto load = [&](int i) { held[i].load(q + i * 16 * (BLOCK_BYTES / 16), sc + i * 16 * (BLOCK / GROUP)); };
  auto advance = [&]() {
    load_b += kw;
    if (load_b < a.blocks) {
      q += kw * (TILE_WORDS / 4);
      sc += kw * (ROWS * BLOCK / GROUP);
    } else if (load_round + 1 < rounds) {
      load_b = part;
      ++load_round;
      begin();
    }  // behind the last block of all it stays where it is, and loads that once more
    if (lane == 0) {  // whose q and sc are where the tile begins
      pesti_umma::l2_prefetch(q, TILE_WORDS * 4);
      pesti_umma::l2_prefetch(sc, ROWS * (BLOCK / GROUP) * 2);
    }
  };
  begin();
#pragma unroll
  for (int i = 0; i < 4; ++i) load(i);
  advance();

  if (sizeof(T) == 4) {
    if (threadIdx.x < 8) most[threadIdx.x] = 0.0f;
    __syncthreads();
    for (int c = 0; c < columns; ++c) {
      float m = 0.0f;
      for (int e = threadIdx.x; e < a.blocks * 16; e += WARPS * 32) {
        EightX<T> v;
        v.load((const T*)a.x + c * a.x_ld, 8 * e, a.D, a.x_vec);
        m = fmaxf(m, v.most());
      }
      m = warp_reduce_fmax(m);
      if (lane == 0) atomicMax((int*)&most[c], __float_as_int(m));  // (not negative)
    }
    __syncthreads();
  }
  for (int c = 0; c < columns; ++c) {
    const float2 up = row_scale(sizeof(T) == 4 ? most[c] : 0.0f, false);
    for (int e = threadIdx.x; e < a.blocks * 16; e += WARPS * 32) {
      EightX<T> v;
      uint4 f[P];
      v.load((const T*)a.x + c * a.x_ld, 8 * e, a.D, a.x_vec);  // block, j, t
      v.template fragments<false>(up, f);
#pragma unroll
      for (int p = 0; p < P; ++p) xs[((e >> 2) * P + p) * columns * 4 + c * 4 + (e & 3)] = f[p];
    }
  }
  if (threadIdx.x == 0) xs[a.blocks * per_block] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  // the lane's fragments; columns without a row read the zeros behind x
  const bool there = g < columns;
  const uint4* mine = there ? xs + g * 4 + t : xs + a.blocks * per_block;
  const int x_block = there ? per_block : 0, x_step = there ? 4 * columns : 0;

  for (int r = 0; r < rounds; ++r) {
    float acc[4][4] = {};
    for (int b = part; b < a.blocks; b += kw) {
      uint4 f[4][P];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int p = 0; p < P; ++p) f[j][p] = mine[b * x_block + (j * P + p) * x_step];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // 16 rows
        const Weights<GROUP>& w = held[i];
#pragma unroll
        for (int gr = 0; gr < BLOCK / GROUP; ++gr) {
          float sum[4];
#pragma unroll
          for (int jj = 0; jj < GROUP / 32; ++jj) {
            const int j = gr * (GROUP / 32) + jj;
            uint32_t q0[4], q1[4];
            unpack<BF16>(((const uint32_t*)&w.w[0])[j], q0);
            unpack<BF16>(((const uint32_t*)&w.w[1])[j], q1);
            const uint32_t fa[2][4] = {{q0[0], q1[0], q0[1], q1[1]}, {q0[2], q1[2], q0[3], q1[3]}};
#pragma unroll
            for (int p = 0; p < P; ++p) {
              if (jj == 0 && p == 0)
                mma<BF16, false>(sum, fa[0], f[j][p].x, f[j][p].y);
              else
                mma<BF16, true>(sum, fa[0], f[j][p].x, f[j][p].y);
              mma<BF16, true>(sum, fa[1], f[j][p].z, f[j][p].w);
            }
          }
          const float s0 = w.scale(0, gr), s1 = w.scale(1, gr);
          acc[i][0] = fmaf(s0, sum[0], acc[i][0]);
          acc[i][1] = fmaf(s0, sum[1], acc[i][1]);
          acc[i][2] = fmaf(s1, sum[2], acc[i][2]);
          acc[i][3] = fmaf(s1, sum[3], acc[i][3]);
        }
        load(i);
      }
      advance();
    }
    const int stack = stack_of(r);
    if (kw > 1) {  // [slot][part - 1][value][lane]; only the part that joins waits for the others
      const int threads = kw * 32;
      if (part) {
        if (r) named_sync(8 + slot, threads);  // the last round's sums are read
        float* to = sums + (slot * (kw - 1) + (part - 1)) * 16 * 32 + lane;
#pragma unroll
        for (int e = 0; e < 16; ++e) to[e * 32] = acc[e >> 2][e & 3];
        named_arrive(1 + slot, threads);
      } else {
        named_sync(1 + slot, threads);
        for (int k = 0; k < kw - 1; ++k)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            acc[e >> 2][e & 3] += sums[((slot * (kw - 1) + k) * 16 + e) * 32 + lane];
        if (r + 1 < rounds) named_arrive(8 + slot, threads);
      }
    }
    if (part || stack >= a.stacks) continue;
    float2 down[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) down[e] = row_scale(sizeof(T) == 4 && 2 * t + e < a.rows ? most[2 * t + e] : 0.0f, true);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int c = 2 * t + (e & 1), v = stack * ROWS + (e >> 2) * 16 + 8 * (e >> 1 & 1) + g;
      if (c < a.rows && v < a.V) store_logit(a, c, v, acc[e >> 2][e & 3] * down[e & 1].x * down[e & 1].y);
    }
  }
}

// --- more rows: products on the tensor cores' own memory
//
// A product's 128 x 128 operand of weights is unpacked into tensor memory as q s, which f16 holds exactly: q has three
// bits beside its sign (or is a power of two) and s eight, once the scales of a part (a few blocks) of a row are brought
// to the right magnitude by a power of two.  Scales below 2^-25 of a part's largest lose bits, which is 2^-35 of what
// that one's weights amount to.  x comes from shared memory.  The sums of a part come back times the inverse power, into
// registers, where a thread adds up one row of the weight for all rows of x.  Tensor memory is read at some 60 bytes a
// clock and SM: taking each group's sums out, to scale them there, bound 48 rows to 107 us (128256 x 4096).  And parts
// keep the tensor cores' sums short, which are cut off and not rounded every 16 of K.

// Blocks of a part: 64 products of 16 of K into one sum, off by up to 6e-7 of it then.
__host__ __device__ constexpr int part_of(int pieces) { return 4 / pieces; }

// x as the products' second operand, [blocks][2][pieces][columns][128 bytes]: half a block's 64 columns in the order
// that words of weights unpack in, 16-byte chunks exchanged as 128-byte swizzled atoms hold them; behind it the rows'
// inverse powers of two.  A block a row.
template <typename T>
__global__ void __launch_bounds__(256) q4_operand_kernel(const LogitArgs a, int columns) {
  pesti_umma::depend_wait();
  pesti_umma::depend_launch();
  constexpr int P = pieces<T>;
  constexpr bool SCALED = scaled<T, true>;
  __shared__ float scratch[33];
  const int n = blockIdx.x, chunks = a.blocks * 16;
  const T* row = (const T*)a.x + n * a.x_ld;
  const bool there = n < a.rows;
  float most = 0.0f;
  if (SCALED) {
    for (int e = threadIdx.x; there && e < chunks; e += 256) {
      EightX<T> v;
      v.load(row, 8 * e, a.D, a.x_vec);
      most = fmaxf(most, v.most());
    }
    most = block_reduce_max(most, scratch);
  }
  const float2 up = row_scale(most, false);
  for (int e = threadIdx.x; e < chunks; e += 256) {
    EightX<T> v;
    uint4 f[P] = {};
    if (there) {
      v.load(row, 8 * e, a.D, a.x_vec);
      v.template fragments<true>(up, f);
    }
#pragma unroll
    for (int p = 0; p < P; ++p)
      a.operand[((long long)((e >> 3) * P + p) * columns + n) * 8 + ((e & 7) ^ (n & 7))] = f[p];
  }
  if (threadIdx.x == 0) ((float2*)(a.operand + (long long)chunks * P * columns))[n] = row_scale(most, true);
}

// A row's scales of a part, as they are held, and the power of two that brings the largest below 2^11 (q s below 2^15).
template <int GROUP, int PART>
struct PartScales {
  uint2 s[PART];  // up to four bf16 a block

  __device__ __forceinline__ void load(const __nv_bfloat16* scales, int b, int blocks) {
#pragma unroll
    for (int i = 0; i < PART; ++i) {
      s[i] = make_uint2(0, 0);
      if (b + i >= blocks) continue;
      const __nv_bfloat16* p = scales + (long long)(b + i) * (ROWS * BLOCK / GROUP);
      if constexpr (GROUP == 32)
        s[i] = __ldg((const uint2*)p);
      else if constexpr (GROUP == 64)
        s[i].x = __ldg((const uint32_t*)p);
      else
        s[i].x = __ldg((const uint16_t*)p);
    }
  }

  __device__ __forceinline__ float at(int block, int g) const {
    const uint32_t v = g < 2 ? s[block].x : s[block].y;
    return bitsf(g & 1 ? v & 0xffff0000u : v << 16);
  }

  // The exponent of that power.
  __device__ __forceinline__ int shift() const {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < PART; ++i)
#pragma unroll
      for (int g = 0; g < BLOCK / GROUP; ++g) most = max(most, fbits(at(i, g)) & 0x7fffffffu);
    const int e = (int)(most >> 23);  // (255: a scale that is NaN, which makes all of the row's sums NaN)
    return min(126, 127 + 10 - e);
  }
};

__device__ __forceinline__ float power(int e) { return bitsf((uint32_t)(e + 127) << 23); }

// Nibbles i and i + 4 of a word as two f16 values q s, in one product: a nibble becomes the four highest bits of 16's
// mantissa, 16 + q + 8, and minus = -24 s, which has 8 + 2 bits and is exact as s is; so is q s.  (q first, then times s,
// by products and sums of two: 86, 99 and 102 us of the kernel below.)
__device__ __forceinline__ void unpack_scaled(uint32_t word, __half2 s, __half2 minus, uint32_t (&q)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = masked(i == 0 ? word << 6 : i == 1 ? word << 2 : i == 2 ? word >> 2 : word >> 6, 0x03c003c0u, 0x4c004c00u);
    const __half2 r = __hfma2(*(const __half2*)&v, s, minus);
    q[i] = *(const uint32_t*)&r;
  }
}

constexpr int WIDE = 128;                       // rows of the weight, two tiles
constexpr int SLOTS = 2;                        // of them at once
constexpr int WIDE_THREADS = (9 * SLOTS + 1) * 32;
constexpr int WIDE_BYTES = WIDE * BLOCK_BYTES;  // of a block

// Where a slot's buffers are in tensor memory: two blocks of unpacked weights, and two parts' sums.
__device__ __forceinline__ uint32_t a_column(int slot, int buf) { return slot * 256 + buf * 64; }
__device__ __forceinline__ uint32_t d_column(int slot, int buf) { return slot * 256 + 128 + buf * 64; }

// Warps 0 to 7 unpack (four a slot, a quarter of the rows each), 8 to 15 add up, 16 copies, 17 and 18 issue a slot's
// products.  128256 x 4096, g 64, f16: 81 us for 16 rows, 95 to 97 for 48, 102 to 112 for 64.  15 or so of them are the packed
// f16 arithmetic that unpacks (64, 81 and 87 without it, of 80, 95 and 98; half of the products would save 1; twice as many
// warps that unpack take 5 more); the weight's bytes would take 43, and what holds the rest is not known.
template <int P, int GROUP, int COLUMNS>
__global__ void __launch_bounds__(WIDE_THREADS, 1) q4_wide_kernel(const LogitArgs a) {
  using namespace pesti_umma;
  constexpr int PART = part_of(P);
  constexpr uint32_t x_half = COLUMNS * 128, x_bytes = 2 * P * x_half, stage = SLOTS * WIDE_BYTES + x_bytes;
  extern __shared__ char raw[];
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  __shared__ uint64_t bars[16 + 8 * SLOTS];
  __shared__ uint32_t tmem_base;
  __shared__ volatile int lost;  // a warp that unpacks gave up
  const uint32_t full = smem_addr(bars), empty = full + 64, a_full = empty + 64, a_empty = a_full + 16 * SLOTS,
                 d_full = a_empty + 16 * SLOTS, d_empty = d_full + 16 * SLOTS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    lost = 0;
    for (int s = 0; s < a.stages; ++s) {
      bar_init(full + 8 * s, 1);
      bar_init(empty + 8 * s, 5 * SLOTS);  // read by the warps that unpack, and its products done
    }
    for (int s = 0; s < 2 * SLOTS; ++s) {
      bar_init(a_full + 8 * s, 4);
      bar_init(a_empty + 8 * s, 1);
      bar_init(d_full + 8 * s, 1);
      bar_init(d_empty + 8 * s, 4);
    }
    bar_init_fence();
  }
  if (warp == 17) tmem_alloc<1>(smem_addr(&tmem_base), 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base;
  depend_wait();
  depend_launch();

  const int per_round = gridDim.x * SLOTS, rounds = (a.stacks + per_round - 1) / per_round;
  auto stack_of = [&](int round, int slot) { return round * per_round + slot * (int)gridDim.x + (int)blockIdx.x; };
  // the scales of the thread's row in a stack
  auto scales_of = [&](int stack) {
    const int v = stack * WIDE + (warp & 3) * 32 + lane;
    return a.scale + (tile_of(min(v, a.V - 1), a.blocks, 0) * ROWS + (v & 63)) * (BLOCK / GROUP);
  };

  if (warp < 4 * SLOTS) {  // unpacks
    const int slot = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t quarter = (uint32_t)(warp & 3) << 21;
    int s = 0, ph = 0, buf = 0, buf_ph = 0;
    // A lane whose wait gives up goes on with the others, so that none part at a tensor memory instruction (a vote on each
    // wait took 5 us more than the 80 for 16 rows), but waits no more and marks what its slots have left as lost.
    bool ok = true;
    for (int r = 0; r < rounds; ++r) {
      const bool there = stack_of(r, slot) < a.stacks;
      const __nv_bfloat16* scales = scales_of(min(stack_of(r, slot), a.stacks - 1));
      PartScales<GROUP, PART> next;
      next.load(scales, 0, a.blocks);
      for (int b0 = 0; b0 < a.blocks; b0 += PART) {
        const PartScales<GROUP, PART> now = next;
        next.load(scales, b0 + PART, a.blocks);
        const float up = power(now.shift());
#pragma unroll
        for (int i = 0; i < PART; ++i) {
          if (b0 + i >= a.blocks) break;
          ok = ok && bar_wait(full + 8 * s, ph);
          uint4 w[4];
          const uint32_t at = base + s * stage + slot * WIDE_BYTES + row * BLOCK_BYTES;
#pragma unroll
          for (int t = 0; t < 4; ++t)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[t].x), "=r"(w[t].y), "=r"(w[t].z), "=r"(w[t].w)
                         : "r"(at + (chunk_at(row, t) << 4)));
          __syncwarp();
          if (lane == 0 && ok) bar_arrive(empty + 8 * s);
          if (++s == a.stages) {
            s = 0;
            ph ^= 1;
          }
          if (!there) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[32];
#pragma unroll
            for (int j = 2 * h; j < 2 * h + 2; ++j) {
              const __half2 scale = __float2half2_rn(now.at(i, j * 32 / GROUP) * up), minus = __hmul2(scale, __float2half2_rn(-24.0f));
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                uint32_t q[4];
                unpack_scaled(((const uint32_t*)&w[t])[j], scale, minus, q);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[16 * (j & 1) + 4 * t + e] = q[e];
              }
            }
            if (h == 0) {
              ok = ok && bar_wait(a_empty + 8 * (2 * slot + buf), buf_ph ^ 1);
              fence_after();
            }
            tmem_store32(tmem + a_column(slot, buf) + 32 * h + quarter, v);
          }
          if (!ok) lost = 1;
          tmem_store_wait();
          fence_before();
          __syncwarp();
          if (lane == 0 && ok) bar_arrive(a_full + 8 * (2 * slot + buf));
          buf ^= 1;
          if (buf == 0) buf_ph ^= 1;
        }
      }
    }
  } else if (warp < 8 * SLOTS) {  // adds up
    const int slot = (warp - 4 * SLOTS) >> 2;
    const uint32_t quarter = (uint32_t)(warp & 3) << 21;
    int buf = 0, buf_ph = 0;
    bool ok = true;  // once a lane's wait has given up, its rows from there on are NaN, without more waiting
    for (int r = 0; r < rounds; ++r) {
      const int stack = stack_of(r, slot);
      if (stack >= a.stacks) break;
      const __nv_bfloat16* scales = scales_of(stack);
      float acc[COLUMNS];
#pragma unroll
      for (int c = 0; c < COLUMNS; ++c) acc[c] = 0.0f;
      for (int b0 = 0; b0 < a.blocks; b0 += PART) {
        PartScales<GROUP, PART> now;
        now.load(scales, b0, a.blocks);
        const float down = power(-now.shift());
        ok = ok && bar_wait(d_full + 8 * (2 * slot + buf), buf_ph) && r != a.give_up;
        fence_after();
        const uint32_t from = tmem + d_column(slot, buf) + quarter;
#pragma unroll
        for (int c = 0; c < COLUMNS; c += 16) {
          uint32_t sum[16];
          tmem_load16(from + c, sum);
          tmem_load_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[c + i] = fmaf(down, bitsf(sum[i]), acc[c + i]);
        }
        fence_before();
        __syncwarp();
        if (lane == 0 && ok) bar_arrive(d_empty + 8 * (2 * slot + buf));
        buf ^= 1;
        if (buf == 0) buf_ph ^= 1;
      }
      ok = ok && !lost;
      const int v = stack * WIDE + (warp & 3) * 32 + lane;
      if (v < a.V) {
        const float2* back = (const float2*)((const char*)a.operand + (long long)a.blocks * x_bytes);
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c)
          if (c < a.rows) store_logit(a, c, v, ok ? acc[c] * back[c].x * back[c].y : NAN);
      }
    }
  } else if (warp == 8 * SLOTS) {  // copies
    if (elect_one()) {
      const int tiles = (a.V + ROWS - 1) / ROWS;
      int s = 0, ph = 0;
      bool ok = true;
      for (int r = 0; r < rounds && ok; ++r) {
        int there = 0;  // tiles of this round's stacks
        for (int slot = 0; slot < SLOTS; ++slot) there += max(0, min(2, tiles - 2 * stack_of(r, slot)));
        for (int b = 0; b < a.blocks; ++b) {
          if (!(ok = bar_wait(empty + 8 * s, ph ^ 1))) break;
          const uint32_t to = base + s * stage;
          bar_expect(full + 8 * s, there * (WIDE_BYTES / 2) + x_bytes);
          for (int i = 0; i < there; ++i) {
            const long long tile = (long long)(2 * stack_of(r, i >> 1) + (i & 1)) * a.blocks + b;
            bulk_load(to + i * (WIDE_BYTES / 2), (const char*)a.q + tile * (WIDE_BYTES / 2), full + 8 * s, WIDE_BYTES / 2);
          }
          bulk_load(to + SLOTS * WIDE_BYTES, (const char*)a.operand + (long long)b * x_bytes, full + 8 * s, x_bytes);
          if (++s == a.stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      for (int i = 0, at = s, at_ph = ph; i < a.stages && ok; ++i) {  // every stage is read
        ok = bar_wait(empty + 8 * at, at_ph ^ 1);
        if (++at == a.stages) {
          at = 0;
          at_ph ^= 1;
        }
      }
      if (!ok)
        for (int i = 0; i < a.stages; ++i) bar_wait(full + 8 * i, i < s ? ph : ph ^ 1);  // copies in flight
    }
  } else {  // issues a slot's products; the warp runs through as one, so that addresses are uniform
    constexpr uint32_t desc = mma_desc(false, false, false, WIDE, COLUMNS);
    const int slot = __shfl_sync(PESTI_FULL_MASK, warp, 0) - (8 * SLOTS + 1);
    int s = 0, ph = 0, abuf = 0, a_ph = 0, dbuf = 0, d_ph = 0;
    bool ok = true;
    for (int r = 0; r < rounds && ok; ++r) {
      const bool there = stack_of(r, slot) < a.stacks;
      for (int b = 0; b < a.blocks && ok; ++b) {
        ok = __all_sync(PESTI_FULL_MASK, bar_wait(full + 8 * s, ph));
        if (ok && there) ok = __all_sync(PESTI_FULL_MASK, bar_wait(a_full + 8 * (2 * slot + abuf), a_ph));
        if (ok && there && b % PART == 0)
          ok = __all_sync(PESTI_FULL_MASK, bar_wait(d_empty + 8 * (2 * slot + dbuf), d_ph ^ 1));
        if (!ok) break;
        if (!there) {  // nothing of this stage is this slot's
          if (lane == 0) bar_arrive(empty + 8 * s);
        } else {
          fence_after();
          const bool last = b % PART == PART - 1 || b == a.blocks - 1;
          if (elect_one()) {
            const uint32_t d = tmem + d_column(slot, dbuf), from = tmem + a_column(slot, abuf);
            const uint64_t xd = operand_desc(base + s * stage + SLOTS * WIDE_BYTES, 0);
#pragma unroll
            for (int k = 0; k < BLOCK; k += 16)
#pragma unroll
              for (int p = 0; p < P; ++p)
                mma_f16_tmem(d, from + k / 2, xd + ((k / 64 * P + p) * x_half >> 4) + k % 64 / 8, desc,
                             b % PART || k || p);
            mma_commit<1>(a_empty + 8 * (2 * slot + abuf));
            mma_commit<1>(empty + 8 * s);
            if (last) mma_commit<1>(d_full + 8 * (2 * slot + dbuf));
          }
          __syncwarp();
          if (last) {
            dbuf ^= 1;
            if (dbuf == 0) d_ph ^= 1;
          }
          abuf ^= 1;
          if (abuf == 0) a_ph ^= 1;
        }
        if (++s == a.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 17) tmem_free<1>(tmem, 512);
}

}  // namespace pesti_q4
