// rowvec.h -- 16-byte chunks of fp32 / bf16 / fp16 rows of any length and alignment, and the 8-bit group form of
// activations, for layer_norm.hip and act8.hip.
#pragma once
#include "common.h"

namespace rv {

struct bf16 { unsigned short u; };
struct fp16 { unsigned short u; };

typedef float f2v __attribute__((ext_vector_type(2)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));

// Rows of an odd number of 2-byte values start at any even address: global memory takes 16-byte accesses at any
// alignment on gfx950 (unaligned access mode is on for HSA), and the type says so to the compiler.
struct __attribute__((packed, aligned(2))) u4_any { unsigned x, y, z, w; };
struct __attribute__((packed, aligned(2))) u2_any { unsigned x, y; };

template <typename T> struct traits;
template <> struct traits<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ void unpack(const u4_any& r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ u4_any pack(const float (&v)[4]) {
    return u4_any{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  }
  static __device__ __forceinline__ float load1(const float* p) { return *p; }
  static __device__ __forceinline__ void store1(float* p, float v) { *p = v; }
};
template <> struct traits<bf16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ void unpack(const u4_any& r, float (&v)[8]) {
    v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
    v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
    v[4] = __uint_as_float(r.z << 16); v[5] = __uint_as_float(r.z & 0xffff0000u);
    v[6] = __uint_as_float(r.w << 16); v[7] = __uint_as_float(r.w & 0xffff0000u);
  }
  static __device__ __forceinline__ unsigned p2(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2v{a, b}), b2v));
  }
  static __device__ __forceinline__ u4_any pack(const float (&v)[8]) {
    return u4_any{p2(v[0], v[1]), p2(v[2], v[3]), p2(v[4], v[5]), p2(v[6], v[7])};
  }
  static __device__ __forceinline__ float load1(const bf16* p) { return __uint_as_float((unsigned)p->u << 16); }
  static __device__ __forceinline__ void store1(bf16* p, float v) {
    p->u = __builtin_bit_cast(unsigned short, (__bf16)v);
  }
};
template <> struct traits<fp16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ void u2(unsigned r, float& a, float& b) {
    const h2v h = __builtin_bit_cast(h2v, r);
    a = (float)h[0];
    b = (float)h[1];
  }
  static __device__ __forceinline__ void unpack(const u4_any& r, float (&v)[8]) {
    u2(r.x, v[0], v[1]); u2(r.y, v[2], v[3]); u2(r.z, v[4], v[5]); u2(r.w, v[6], v[7]);
  }
  // round to nearest even (v_cvt_f16_f32; the packed conversion of this width would round to zero)
  static __device__ __forceinline__ unsigned p2(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2v{a, b}), h2v));
  }
  static __device__ __forceinline__ u4_any pack(const float (&v)[8]) {
    return u4_any{p2(v[0], v[1]), p2(v[2], v[3]), p2(v[4], v[5]), p2(v[6], v[7])};
  }
  static __device__ __forceinline__ float load1(const fp16* p) { return (float)__builtin_bit_cast(_Float16, p->u); }
  static __device__ __forceinline__ void store1(fp16* p, float v) {
    p->u = __builtin_bit_cast(unsigned short, (_Float16)v);
  }
};

// One chunk of a row: `left` = values from p to the row's end (may be <= 0: zeros).  The whole chunk is one 16-byte load;
// the last, partial chunk of a row is read value by value and never past the end.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* __restrict__ p, int left, float (&v)[traits<T>::VEC]) {
  constexpr int VEC = traits<T>::VEC;
  if (left >= VEC) {
    traits<T>::unpack(*reinterpret_cast<const u4_any*>(p), v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = 0.f;
    if (left > 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float f = traits<T>::load1(p + (i < left ? i : 0));
        v[i] = i < left ? f : 0.f;
      }
    }
  }
}
// `room` = values from p to the end of what may be written
template <typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ p, int room, const float (&v)[traits<T>::VEC]) {
  constexpr int VEC = traits<T>::VEC;
  if (room >= VEC) {
    *reinterpret_cast<u4_any*>(p) = traits<T>::pack(v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < room) traits<T>::store1(p + i, v[i]);
  }
}

// ---------------------------------------------------------------------------------------------- 8-bit group form
// 32 consecutive channels of a row (the last group of a row may be shorter) share a power of two 2^e; a value is held as
// int8 code = rint(x 2^-e).  e is the smallest exponent >= -126 with rint(absmax 2^-e) <= 127: with absmax = 1.f 2^p
// that is p - 6, and one more where 1.f >= 127.5 / 64, i.e. the mantissa field >= 0x7f0000 -- adding 0x10000 to the bit
// pattern carries into the exponent field exactly then.  At the end of the range e stays 121 and codes stop at 127 (128 2^121
// is no finite fp32).  Held as the biased exponent e + 127 in 1 .. 248; a group with an
// infinity or a NaN holds 255 and codes 0: 0 x 2^128 (= inf as fp32 bits) is NaN, so all its values come back as NaN.
// Every held value has 7 significant bits and a bf16 exponent: code 2^e is exact in bf16 (and fp32).
constexpr int GROUP = 32;

__device__ __forceinline__ unsigned group_scale(unsigned absmax_bits) {
  const int e = (int)((absmax_bits + 0x10000u) >> 23) - 6;
  return absmax_bits >= 0x7f800000u ? 255u : (unsigned)min(max(e, 1), 248);
}
// 2^-e as fp32 (0 for a non-finite group: its codes are set to zero by group_code)
__device__ __forceinline__ float group_inverse(unsigned scale) {
  return scale == 255u ? 0.f : __uint_as_float((254u - scale) << 23);
}
__device__ __forceinline__ float group_step(unsigned scale) { return __uint_as_float(scale << 23); }
__device__ __forceinline__ int group_code(float x, float inverse) {
  return inverse == 0.f ? 0 : (int)fminf(fmaxf(rintf(x * inverse), -127.f), 127.f);
}
// four codes, 2^e -> four values (exact; scale 255: 0 x inf = NaN)
__device__ __forceinline__ void group_values(unsigned codes, float step, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)(signed char)(codes >> (8 * i)) * step;
}

template <int VEC>
__device__ __forceinline__ void load_codes(const signed char* __restrict__ p, float step, float (&v)[VEC]) {
  if (VEC == 8) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    float a[4], b[4];
    group_values(r.x, step, a);
    group_values(r.y, step, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[VEC / 2 + i] = b[i]; }
  } else {
    float a[4];
    group_values(*reinterpret_cast<const unsigned*>(p), step, a);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i];
  }
}

// The scale of this lane's group: LANES consecutive lanes (a power of two) hold the group's values, VEC each
template <int VEC, int LANES>
__device__ __forceinline__ unsigned lanes_scale(const float (&v)[VEC]) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < VEC; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);   // as integers: NaN is the largest
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
  return group_scale(m);
}
template <int VEC>
__device__ __forceinline__ void store_codes(signed char* __restrict__ p, const float (&v)[VEC], float inverse) {
  unsigned w[VEC / 4];
#pragma unroll
  for (int q = 0; q < VEC / 4; ++q) {
    w[q] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[q] |= ((unsigned)group_code(v[q * 4 + i], inverse) & 0xffu) << (8 * i);
  }
  if (VEC == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[VEC / 4 - 1]);
  else
    *reinterpret_cast<unsigned*>(p) = w[0];
}

}  // namespace rv
