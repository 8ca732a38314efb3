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

// Tensors that no cache holds until their next use are read and written past the caches (non-temporal): from STREAM_BYTES
// on, as instances of their own (a choice at run time cost more than it gave).  bf16: forward 1572864 x 64 73.7 us, so 68.4;
// backward 786432 x 128 117.5, 106; forward and backward with 8 bits kept, 393216 x 196 186, 165.5; pack and unpack
// 786432 x 96 77.7, 71.  The next kernel counts too.  With the chain's consumers (rows of 128 bf16 channels; cached, past the caches, us):
//                                       33 MB   67 MB         100 MB        134 MB        201 MB        402 MB
//   forward, then the next product      35, 38  58.3, 61.8    78.4, 84.9    106.7, 109.6  163.8, 161.1  317.9, 315.1
//   forward, product, packing           44, 48  73.8, 76.5    104.3, 107.6  140.9, 143.6  215.9, 216.0  426.0, 426.6
//   product, backward, product          68, 69  105.8, 110.0  148.1, 151.7  202.8, 193.8  306.0, 285.8  582.5, 557.5
// The forward alone would change over a little later, the two passes together do so here.
constexpr long long STREAM_BYTES = 1ll << 27;
typedef unsigned v4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned v2_any __attribute__((ext_vector_type(2), aligned(2)));
template <bool STREAM>
__device__ __forceinline__ void put(void* p, const u4_any& r) {
  if (STREAM) __builtin_nontemporal_store(v4_any{r.x, r.y, r.z, r.w}, reinterpret_cast<v4_any*>(p));
  else *reinterpret_cast<u4_any*>(p) = r;
}
template <bool STREAM>
__device__ __forceinline__ void put(void* p, const u2_any& r) {
  if (STREAM) __builtin_nontemporal_store(v2_any{r.x, r.y}, reinterpret_cast<v2_any*>(p));
  else *reinterpret_cast<u2_any*>(p) = r;
}
template <bool STREAM>
__device__ __forceinline__ void get(const void* p, u4_any& r) {
  if (STREAM) {
    const v4_any v = __builtin_nontemporal_load(reinterpret_cast<const v4_any*>(p));
    r = u4_any{v[0], v[1], v[2], v[3]};
  } else {
    r = *reinterpret_cast<const u4_any*>(p);
  }
}
template <bool STREAM>
__device__ __forceinline__ void get(const void* p, u2_any& r) {
  if (STREAM) {
    const v2_any v = __builtin_nontemporal_load(reinterpret_cast<const v2_any*>(p));
    r = u2_any{v[0], v[1]};
  } else {
    r = *reinterpret_cast<const u2_any*>(p);
  }
}

template <typename T, bool STREAM>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&v)[traits<T>::VEC]) {
  put<STREAM>(p, traits<T>::pack(v));
}

// base + offset in bytes, base the same for the whole wave: one 32-bit register per lane for the address
template <typename P>
__device__ __forceinline__ P* at32(P* base, unsigned bytes) {
  return (P*)((const char*)base + bytes);        // (pointer arithmetic: through an integer the access would be a flat one)
}

// A lane's chunk of a row of C >= VEC values: whole chunks start at c, a multiple of VEC; the last, partial one is taken as
// the row's last VEC values instead -- it overlaps its neighbour by `skip` values, which this lane computes a second time
// (the same bits) and leaves out of every sum.  So all loads and stores are whole and unconditional: a guarded load is a
// branch, and the loads behind it wait for the ones before.  A lane behind the row's end (c >= C) owns nothing.
template <int VEC>
struct window {
  int c, at, skip;
  __device__ __forceinline__ window(int c_, int C) : c(c_), at(min(c_, C - VEC)), skip(min(c_ - min(c_, C - VEC), VEC)) {}
};

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
__device__ __forceinline__ float group_inverse(unsigned scale) { return __uint_as_float((254u - min(scale, 248u)) << 23); }
__device__ __forceinline__ float group_step(unsigned scale) { return __uint_as_float(scale << 23); }

// VEC codes, four to a word.  x 2^-e is exact and at most 127.5, so adding 1.5 2^23 leaves its integer part, rounded to
// nearest even, in the low byte of the sum's bit pattern, two's complement.  Only the last scale needs codes held at 127 and
// only 255 codes set to zero: one branch for a wave that has either.
template <int VEC>
__device__ __forceinline__ void group_codes(const float (&v)[VEC], unsigned scale, unsigned (&w)[VEC / 4]) {
  const float inverse = group_inverse(scale);
  unsigned t[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) t[i] = __float_as_uint(fmaf(v[i], inverse, 12582912.f));
  if (__any(scale >= 248u)) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      t[i] = scale == 255u ? 0u : __float_as_uint(fminf(fmaxf(v[i] * inverse, -127.f), 127.f) + 12582912.f);
  }
#pragma unroll
  for (int q = 0; q < VEC / 4; ++q)
    w[q] = __builtin_amdgcn_perm(t[4 * q + 1], t[4 * q], 0x0c0c0400u) | __builtin_amdgcn_perm(t[4 * q + 3], t[4 * q + 2], 0x04000c0cu);
}
// a window's codes to their place: the values it skips are a neighbour's
__device__ __forceinline__ void store_codes(signed char* __restrict__ p, int skip, const unsigned (&w)[2]) {
  const unsigned long long b = (((unsigned long long)w[1] << 32) | w[0]) >> (8 * (skip & 7));
  *reinterpret_cast<uint2*>(p) = make_uint2((unsigned)b, (unsigned)(b >> 32));
}
__device__ __forceinline__ void store_codes(signed char* __restrict__ p, int skip, const unsigned (&w)[1]) {
  *reinterpret_cast<unsigned*>(p) = w[0] >> (8 * (skip & 3));
}
// the codes of a window, at any alignment
struct __attribute__((packed, aligned(1))) u2_byte { unsigned x, y; };
struct __attribute__((packed, aligned(1))) u1_byte { unsigned x; };
__device__ __forceinline__ void load_codes(const signed char* __restrict__ p, unsigned (&w)[2]) {
  const u2_byte r = *reinterpret_cast<const u2_byte*>(p);
  w[0] = r.x;
  w[1] = r.y;
}
__device__ __forceinline__ void load_codes(const signed char* __restrict__ p, unsigned (&w)[1]) {
  w[0] = reinterpret_cast<const u1_byte*>(p)->x;
}
// code i as fp32; times the group's step: the held value (exact; scale 255: 0 x inf = NaN)
template <int N>
__device__ __forceinline__ float code_at(const unsigned (&w)[N], int i) { return (float)(signed char)(w[i >> 2] >> (8 * (i & 3))); }

// ---------------------------------------------------------------------------------------------- across lanes
// Sums and maxima over 2, 4, .. 64 neighbouring lanes, every lane getting the result: the mirrored permutations equal an
// exchange with lane ^ 4 / lane ^ 8 once the smaller groups hold one value each.
__device__ __forceinline__ unsigned dpp(unsigned v, int step) {
  switch (step) {
    case 1: return __builtin_amdgcn_update_dpp(0u, v, 0xB1, 0xf, 0xf, true);       // quad_perm 1 0 3 2
    case 2: return __builtin_amdgcn_update_dpp(0u, v, 0x4E, 0xf, 0xf, true);       // quad_perm 2 3 0 1
    case 4: return __builtin_amdgcn_update_dpp(0u, v, 0x141, 0xf, 0xf, true);      // row_half_mirror
    default: return __builtin_amdgcn_update_dpp(0u, v, 0x140, 0xf, 0xf, true);     // row_mirror
  }
}
// lane ^ 8: a turn by eight within rows of 16 (row_ror:8)
__device__ __forceinline__ unsigned turn8(unsigned v) { return __builtin_amdgcn_update_dpp(0u, v, 0x128, 0xf, 0xf, true); }
// once lanes 8 apart hold the same: a turn by four makes lane ^ 4 of it
__device__ __forceinline__ unsigned turn4(unsigned v) { return __builtin_amdgcn_update_dpp(0u, v, 0x124, 0xf, 0xf, true); }
__device__ __forceinline__ float add16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  if (LANES > 1) v += __uint_as_float(dpp(__float_as_uint(v), 1));
  if (LANES > 2) v += __uint_as_float(dpp(__float_as_uint(v), 2));
  if (LANES > 4) v += __uint_as_float(dpp(__float_as_uint(v), 4));
  if (LANES > 8) v += __uint_as_float(dpp(__float_as_uint(v), 8));
  if (LANES > 16) v = add16(v);
  if (LANES > 32) v = add32(v);
  return v;
}
template <int LANES>                                      // 8 lanes at most
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
  if (LANES > 1) v = max(v, dpp(v, 1));
  if (LANES > 2) v = max(v, dpp(v, 2));
  if (LANES > 4) v = max(v, dpp(v, 4));
  return v;
}

// workgroups for n > 0 passes, `most` at most, all with the same number of passes (but the last few)
static inline unsigned even_grid(long long n, long long most) {
  const long long passes = (n + most - 1) / most;
  return (unsigned)((n + passes - 1) / passes);
}

// ---------------------------------------------------------------------------------------------- partial sums
// out[e] = sum over p of part[p][count], e < count, in a fixed order: SL slices of p a workgroup, 1024 / SL threads across,
// W (1 or 4) columns each, eight loads in flight per thread.  e < first goes to a, the rest to b.
template <int SL, int W>
__global__ __launch_bounds__(1024) void fold_kernel(int P, size_t count, size_t first, const float* __restrict__ part,
                                                    float* __restrict__ a, float* __restrict__ b) {
  constexpr int TX = 1024 / SL;
  constexpr int NP = TX < 64 ? 16 : SL;                    // sums of a column that meet in LDS: a wave's or a slice's
  __shared__ float s[NP][TX * W];
  const int tx = threadIdx.x % TX, sl = threadIdx.x / TX;
  const size_t base = (size_t)blockIdx.x * TX * W, e = base + (size_t)tx * W;
  float v[W];
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] = 0.f;
  auto get = [&](int p, float (&f)[W]) {
    const float* q = part + (size_t)p * count + e;
    if (W == 4) {
      const float4 r = *reinterpret_cast<const float4*>(q);
      f[0] = r.x; f[W > 1 ? 1 : 0] = r.y; f[W > 2 ? 2 : 0] = r.z; f[W > 3 ? 3 : 0] = r.w;
    } else {
      f[0] = *q;
    }
  };
  if (e < count) {
    int i = sl;
    for (; i + 7 * SL < P; i += 8 * SL) {
      float f[8][W];
#pragma unroll
      for (int j = 0; j < 8; ++j) get(i + j * SL, f[j]);
#pragma unroll
      for (int j = 0; j < W; ++j)
        v[j] += ((f[0][j] + f[1][j]) + (f[2][j] + f[3][j])) + ((f[4][j] + f[5][j]) + (f[6][j] + f[7][j]));
    }
    for (; i < P; i += SL) {
      float f[W];
      get(i, f);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] += f[j];
    }
  }
  // slices of a wave in registers, the rest through LDS once
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if (TX == 16) v[j] = add16(v[j]);
    if (TX <= 32) v[j] = add32(v[j]);
  }
  if (TX >= 64 || (threadIdx.x & 63) < TX) {
#pragma unroll
    for (int j = 0; j < W; ++j) s[TX < 64 ? threadIdx.x >> 6 : sl][tx * W + j] = v[j];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < TX * W && base + c < count; c += 1024) {
    float t = s[0][c];
#pragma unroll
    for (int g = 1; g < NP; ++g) t += s[g][c];
    (base + c < first ? a[base + c] : b[base + c - first]) = t;
  }
}
static inline int fold(int P, size_t count, size_t first, const float* part, float* a, float* b, hipStream_t st) {
  // slices: as many as leave a thread about eight partial sums (64 slices of 16 columns still read whole 64-byte lines);
  // four columns a thread for many columns (256 sums of 256 x 128: 7.1 us with 32 slices, 10.0 with 16; 64 sums of
  // 512 x 256 the other way round, 9.0 and 7.4)
#define RV_FOLD(SL, W)                                                                                                    \
  hipLaunchKernelGGL((fold_kernel<SL, W>), dim3((unsigned)((count + W * 1024 / SL - 1) / (W * 1024 / SL))), dim3(1024), 0, \
                     st, P, count, first, part, a, b)
  const bool wide = count >= 32768 && (count & 3) == 0;
  if (wide && P >= 128) RV_FOLD(32, 4);
  else if (wide && P >= 64) RV_FOLD(16, 4);
  else if (wide && P >= 16) RV_FOLD(4, 4);
  else if (wide) RV_FOLD(2, 4);
  else if (P >= 256) RV_FOLD(64, 1);
  else if (P >= 64) RV_FOLD(32, 1);
  else if (P >= 16) RV_FOLD(8, 1);
  else RV_FOLD(2, 1);
#undef RV_FOLD
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace rv
