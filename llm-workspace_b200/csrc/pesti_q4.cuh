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

#include "pesti_common.cuh"

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
  int rows, D, pieces, columns;  // columns = rows * pieces: f32 rows are three bf16 ones
  const uint4* q;
  const __nv_bfloat16* scale;
  int V, blocks;
  uint4* frags;  // [blocks][4][NT][32]
  void* y;
  long long y_ld;
  int out;  // 0 f32, 1 bf16, 2 f16
  int k_warps;
};

// x as the products' fragments: word j of a block and column tile n, lane (column g, t): the pairs that a word of
// weights unpacks to.  f32 is cut into three bf16 whose sum it is, exactly.
template <typename T, int NT>
__global__ void __launch_bounds__(128) q4_fragments_kernel(const LogitArgs a) {
  const int b = blockIdx.x, j = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  for (int n = 0; n < NT; ++n) {
    const int c = n * 8 + g, row = c / a.pieces, piece = c - row * a.pieces;
    uint16_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = b * BLOCK + 32 * j + 8 * t + i;
      v[i] = 0;
      if (row >= a.rows || d >= a.D) continue;
      const T x = ((const T*)a.x)[row * a.x_ld + d];
      if constexpr (sizeof(T) == 2) {
        v[i] = *(const uint16_t*)&x;
      } else {
        float rest = x;
        uint32_t bits = fbits(rest);
        for (int p = 0; p < piece; ++p) {
          const bool whole = (bits & 0x7f800000u) == 0x7f800000u;  // inf and NaN are in the first piece
          rest = whole ? 0.0f : rest - bitsf(bits & 0xffff0000u);
          bits = fbits(rest);
        }
        v[i] = (uint16_t)(bits >> 16);
        if (is_nan(rest)) v[i] |= 0x40;
      }
    }
    uint4 f;
    uint32_t* p = (uint32_t*)&f;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = (uint32_t)v[i] | (uint32_t)v[i + 4] << 16;
    a.frags[((long long)(b * 4 + j) * NT + n) * 32 + lane] = f;
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

constexpr int WARPS = 8;
constexpr int ROWS = 32;  // of the weight, per warp

__device__ __forceinline__ void store_logit(const LogitArgs& a, int row, int v, float y) {
  const long long at = row * a.y_ld + v;
  if (a.out == 0)
    ((float*)a.y)[at] = y;
  else if (a.out == 1)
    ((__nv_bfloat16*)a.y)[at] = __float2bfloat16_rn(y);
  else
    ((__half*)a.y)[at] = __float2half_rn(y);
}

// A warp multiplies 32 rows of the weight by all columns over its share of K; the k_warps warps of a row tile join
// their sums in shared memory, in their order.
template <bool F16, int GROUP, int NT>
__global__ void __launch_bounds__(WARPS * 32) q4_logits_kernel(const LogitArgs a) {
  __shared__ float sums[WARPS][8][ROWS + 1];  // a column tile at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kw = a.k_warps, wr = WARPS / kw, part = warp % kw, tile = warp / kw;
  const int row0 = (blockIdx.x * wr + tile) * ROWS;
  const int b0 = a.blocks * part / kw, b1 = a.blocks * (part + 1) / kw;
  const uint4* q[4];
  const __nv_bfloat16* sc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = min(row0 + g + 8 * i, a.V - 1);
    q[i] = a.q + (row * a.blocks) * (BLOCK_BYTES / 16) + t;
    sc[i] = a.scale + (row * a.blocks) * (BLOCK / GROUP);
  }
  float acc[2][NT][4] = {};
  if (row0 < a.V) {
    for (int b = b0; b < b1; ++b) {
      uint4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __ldcs(q[i] + b * (BLOCK_BYTES / 16));
#pragma unroll
      for (int gr = 0; gr < BLOCK / GROUP; ++gr) {
        float part_acc[2][NT][4] = {};
#pragma unroll
        for (int jj = 0; jj < GROUP / 32; ++jj) {
          const int j = gr * (GROUP / 32) + jj;
          uint32_t word[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) word[i] = ((const uint32_t*)&w[i])[j];
          uint32_t fa[2][2][4];
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              fa[m][h][0] = unpack<F16>(word[2 * m], 2 * h);
              fa[m][h][1] = unpack<F16>(word[2 * m + 1], 2 * h);
              fa[m][h][2] = unpack<F16>(word[2 * m], 2 * h + 1);
              fa[m][h][3] = unpack<F16>(word[2 * m + 1], 2 * h + 1);
            }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 f = a.frags[((long long)(b * 4 + j) * NT + n) * 32 + lane];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              mma<F16>(part_acc[m][n], fa[m][0], f.x, f.y);
              mma<F16>(part_acc[m][n], fa[m][1], f.z, f.w);
            }
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float s0 = __bfloat162float(sc[2 * m][b * (BLOCK / GROUP) + gr]);
          const float s1 = __bfloat162float(sc[2 * m + 1][b * (BLOCK / GROUP) + gr]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[m][n][0] = fmaf(s0, part_acc[m][n][0], acc[m][n][0]);
            acc[m][n][1] = fmaf(s0, part_acc[m][n][1], acc[m][n][1]);
            acc[m][n][2] = fmaf(s1, part_acc[m][n][2], acc[m][n][2]);
            acc[m][n][3] = fmaf(s1, part_acc[m][n][3], acc[m][n][3]);
          }
        }
      }
    }
  }
  // columns of f32 rows do not cross a tile: the host gives them NT * 8 / 3 rows, so tiles are joined one by one
  __shared__ float rest[WARPS][ROWS];  // what a row's pieces before this tile sum to
#pragma unroll 1
  for (int n = 0; n < NT; ++n) {
    __syncthreads();
#pragma unroll
    for (int nn = 0; nn < NT; ++nn) {
      if (nn != n) continue;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        sums[warp][2 * t][16 * m + g] = acc[m][nn][0];
        sums[warp][2 * t + 1][16 * m + g] = acc[m][nn][1];
        sums[warp][2 * t][16 * m + g + 8] = acc[m][nn][2];
        sums[warp][2 * t + 1][16 * m + g + 8] = acc[m][nn][3];
      }
    }
    __syncthreads();
    if (a.pieces == 1) {
      for (int e = threadIdx.x; e < wr * 8 * ROWS; e += WARPS * 32) {
        const int r = e % ROWS, c = e / ROWS % 8, w = e / (8 * ROWS) * kw;
        const int v = (blockIdx.x * wr + w / kw) * ROWS + r;
        if (n * 8 + c >= a.columns || v >= a.V) continue;
        float y = 0.0f;
        for (int k = 0; k < kw; ++k) y += sums[w + k][c][r];
        store_logit(a, n * 8 + c, v, y);
      }
    } else {
      for (int e = threadIdx.x; e < wr * ROWS; e += WARPS * 32) {
        const int r = e % ROWS, w = e / ROWS * kw, v = (blockIdx.x * wr + w / kw) * ROWS + r;
        float y = n ? rest[w][r] : 0.0f;
        for (int c = 0; c < 8 && n * 8 + c < a.columns; ++c) {
          for (int k = 0; k < kw; ++k) y += sums[w + k][c][r];
          if ((n * 8 + c) % 3 == 2) {
            if (v < a.V) store_logit(a, (n * 8 + c) / 3, v, y);
            y = 0.0f;
          }
        }
        rest[w][r] = y;
      }
    }
  }
}

}  // namespace pesti_q4
