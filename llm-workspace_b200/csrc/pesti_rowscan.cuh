// Shared pieces of the kernels that stream whole logit rows (beam selection,
// distillation): a row cut into units that one warp holds in registers, the
// unit's maximum and its sum of exponentials.
//
// A row may start at any element.  It is read in 16-byte vectors of the
// aligned address space: vector j of a row whose first element sits h elements
// behind a 16-byte boundary covers elements [j*VE - h, (j+1)*VE - h).  32
// vectors in a row (one per lane) are a segment, 8 segments a unit: 2048
// 16-bit or 1024 32-bit elements, 4 KB.  Segments are contiguous in the row,
// so their order is the order of the elements.  Vectors that reach over an end
// of the row are read element by element, and hold -inf where there is none.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace pesti_rows {

constexpr int UNIT_VECS = 8;                  // 16-byte vectors per lane and unit
constexpr int UNIT_SLOTS = UNIT_VECS * 32;    // vectors per unit
constexpr uint32_t FULL = 0xffffffffu;

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float pos_inf() { return __int_as_float(0x7f800000); }

// 2^x by the hardware (relative error at most 2^-22.5; 2^0 and 2^-inf exact).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 operations in one instruction (sm_100).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// Maximum over the warp's lanes, NaN lanes left out (sm_100a).
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

template <typename T>
struct Elem;

template <>
struct Elem<float> {
  static constexpr int VE = 4;        // elements of a 16-byte vector
  static constexpr int PAIRS = 2;     // pairs of a vector
  static constexpr uint32_t NEG_INF = 0xff800000u;
  static __device__ __forceinline__ float load(const void* p, long long i) { return ((const float*)p)[i]; }
  static __device__ __forceinline__ void store(void* p, long long i, float v) { ((float*)p)[i] = v; }
  static __device__ __forceinline__ float2 pair(const uint4& v, int q) {
    return q == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ float vec_max(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                 fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ uint32_t bits(const void* p, long long i) { return ((const uint32_t*)p)[i]; }
  // element `sub` of the vector set to the given bits
  static __device__ __forceinline__ void put(uint4& v, int sub, uint32_t b) {
    v.x = sub == 0 ? b : v.x;
    v.y = sub == 1 ? b : v.y;
    v.z = sub == 2 ? b : v.z;
    v.w = sub == 3 ? b : v.w;
  }
  static __device__ __forceinline__ float at(const uint4& v, int e) {
    return __uint_as_float(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ void pack(uint4& v, int q, float2 f) {
    (q == 0 ? v.x : v.z) = __float_as_uint(f.x);
    (q == 0 ? v.y : v.w) = __float_as_uint(f.y);
  }
};

// The two 16-bit types share the vector handling.
template <typename H>
struct Elem16 {
  static constexpr int VE = 8;
  static constexpr int PAIRS = 4;
  static __device__ __forceinline__ uint32_t bits(const void* p, long long i) { return ((const uint16_t*)p)[i]; }
  static __device__ __forceinline__ uint32_t word(const uint4& v, int q) {
    return q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w;
  }
  static __device__ __forceinline__ uint32_t put1(uint32_t w, int sub, int at, uint32_t b) {
    if (sub == at) w = (w & 0xffff0000u) | b;
    if (sub == at + 1) w = (w & 0x0000ffffu) | (b << 16);
    return w;
  }
  static __device__ __forceinline__ void put(uint4& v, int sub, uint32_t b) {
    v.x = put1(v.x, sub, 0, b);
    v.y = put1(v.y, sub, 2, b);
    v.z = put1(v.z, sub, 4, b);
    v.w = put1(v.w, sub, 6, b);
  }
};

template <>
struct Elem<__nv_bfloat16> : Elem16<__nv_bfloat16> {
  static constexpr uint32_t NEG_INF = 0xff80u;
  static __device__ __forceinline__ float load(const void* p, long long i) {
    return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  }
  static __device__ __forceinline__ void store(void* p, long long i, float v) {
    ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  }
  static __device__ __forceinline__ float at(const uint4& v, int e) {
    return __uint_as_float((word(v, e >> 1) >> ((e & 1) * 16)) << 16);
  }
  static __device__ __forceinline__ float2 pair(const uint4& v, int q) {
    const uint32_t w = word(v, q);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ float vec_max(const uint4& v) {
    const __nv_bfloat162 *a = (const __nv_bfloat162*)&v.x, *b = (const __nv_bfloat162*)&v.y,
                         *c = (const __nv_bfloat162*)&v.z, *d = (const __nv_bfloat162*)&v.w;
    const __nv_bfloat162 m = __hmax2(__hmax2(*a, *b), __hmax2(*c, *d));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void pack(uint4& v, int q, float2 f) {
    const __nv_bfloat162 h = __float22bfloat162_rn(f);
    (q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w) = *(const uint32_t*)&h;
  }
};

template <>
struct Elem<__half> : Elem16<__half> {
  static constexpr uint32_t NEG_INF = 0xfc00u;
  static __device__ __forceinline__ float load(const void* p, long long i) {
    return __half2float(((const __half*)p)[i]);
  }
  static __device__ __forceinline__ void store(void* p, long long i, float v) {
    ((__half*)p)[i] = __float2half_rn(v);
  }
  static __device__ __forceinline__ float at(const uint4& v, int e) {
    return __half2float(__ushort_as_half((unsigned short)(word(v, e >> 1) >> ((e & 1) * 16))));
  }
  static __device__ __forceinline__ float2 pair(const uint4& v, int q) {
    const uint32_t w = word(v, q);
    return __half22float2(*(const __half2*)&w);
  }
  static __device__ __forceinline__ float vec_max(const uint4& v) {
    const __half2 *a = (const __half2*)&v.x, *b = (const __half2*)&v.y, *c = (const __half2*)&v.z,
                  *d = (const __half2*)&v.w;
    const __half2 m = __hmax2(__hmax2(*a, *b), __hmax2(*c, *d));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void pack(uint4& v, int q, float2 f) {
    const __half2 h = __float22half2_rn(f);
    (q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w) = *(const uint32_t*)&h;
  }
};

// Elements that row `p` starts behind a 16-byte boundary.
template <typename T>
__host__ __device__ __forceinline__ int row_head(const void* p) {
  return (int)(((uintptr_t)p & 15) / sizeof(T));
}

template <typename T>
__host__ __device__ __forceinline__ long long unit_elems() {
  return (long long)UNIT_SLOTS * (16 / (long long)sizeof(T));
}

// Units of a row of V elements at any alignment (the head adds less than one vector).
template <typename T>
__host__ __device__ __forceinline__ long long row_units(long long V) {
  const long long ve = 16 / (long long)sizeof(T);
  return (V + ve - 1 + unit_elems<T>() - 1) / unit_elems<T>();
}

// One vector of a row, element by element: -inf outside [0, V).
template <typename T>
__device__ __noinline__ uint4 load_edge(const void* row, long long lo, long long V) {
  uint4 r;
  const uint32_t ninf = Elem<T>::NEG_INF;
  r.x = r.y = r.z = r.w = sizeof(T) == 4 ? ninf : (ninf | (ninf << 16));
  for (int e = 0; e < Elem<T>::VE; ++e) {
    const long long i = lo + e;
    if (i >= 0 && i < V) Elem<T>::put(r, e, Elem<T>::bits(row, i));
  }
  return r;
}

// Loads unit u of the row into v (vector i of lane l is vector u*256 + i*32 + l).
// NC: the row is not written while the kernel runs (read-only loads).
template <typename T, bool NC>
__device__ __forceinline__ void load_unit(uint4 (&v)[UNIT_VECS], const T* row, int head, long long V, long long u,
                                          int lane) {
  constexpr int VE = Elem<T>::VE;
  const long long first = u * UNIT_SLOTS * VE - head;  // element of the unit's first slot
  const uint4* base = (const uint4*)(row - head) + u * UNIT_SLOTS + lane;
  if (first >= 0 && first + UNIT_SLOTS * VE <= V) {
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i) v[i] = NC ? __ldg(base + i * 32) : base[i * 32];
  } else {
#pragma unroll
    for (int i = 0; i < UNIT_VECS; ++i) {
      const long long lo = first + (long long)(i * 32 + lane) * VE;
      if (lo >= 0 && lo + VE <= V)
        v[i] = NC ? __ldg(base + i * 32) : base[i * 32];
      else
        v[i] = load_edge<T>(row, lo, V);
    }
  }
}

// References of a unit's or row's sum of 2^(x*c), for the largest x = m:
//  - ordinarily R = ceil(m*c), an integer, so that sums of two references are
//    joined by an exact power of two;
//  - where |m*c| >= 2^30 (masks of the type's lowest value, +inf) the next
//    smaller f32 is more than 44/c * log2(e) below m: every x but m itself
//    vanishes against m, and the sum is the number of x equal to m.  (A caller
//    may set the limit lower.)
constexpr float FAR = 1073741824.0f;
__device__ __forceinline__ bool is_far(float m, float c, float far = FAR) { return !(fabsf(m * c) < far); }

// 2^d for an integer-valued d <= 0 (0 below the range of a double).
__device__ __forceinline__ double pow2i(double d) {
  return d < -1022.0 ? 0.0 : __hiloint2double((int)(1023.0 + d) << 20, 0);
}

// Factor from the reference of m_old to that of m_new >= m_old.
__device__ __forceinline__ double ref_scale(float m_old, float m_new, float c, float far = FAR) {
  if (m_old == m_new) return 1.0;
  if (!(m_old > neg_inf()) || is_far(m_old, c, far) || is_far(m_new, c, far)) return 0.0;
  return pow2i((double)ceilf(m_old * c) - (double)ceilf(m_new * c));
}

}  // namespace pesti_rows
