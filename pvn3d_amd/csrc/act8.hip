// act8.hip -- activations put away in 8 bits for the backward pass, and the weight gradient taken from them (gfx950).
//
// A layer's input is kept for dW = dY^T X only.  Here it is kept in the group form of rowvec.h: int8 codes and one power of
// two per 32 channels of a row, 33/32 bytes per value instead of 2, off by at most half a step of 1/64 to 1/128 of the
// group's largest magnitude.  Every held value is exact in bf16, so the matrix instructions take it without a further
// rounding: dW is the exact product of dY and the held values, summed in fp32.
#include "rowvec.h"

namespace {

using rv::bf16;
using rv::fp16;
using rv::traits;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// ------------------------------------------------------------------------------------------------ pack / unpack
// tpr threads across a row (a power of two that covers whole groups or the row), 256 / tpr rows per workgroup.  Chunks are
// windows (rowvec.h); a row shorter than one is read value by value.
template <typename T>
__device__ __forceinline__ void load_any(const T* __restrict__ row, int at, int C, float (&v)[traits<T>::VEC]) {
  constexpr int VEC = traits<T>::VEC;
  if (C >= VEC) {
    rv::load_vec<T>(row + at, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = i < C ? traits<T>::load1(row + i) : 0.f;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void act8_pack_kernel(long long rows, int C, int tpr, const T* __restrict__ x,
                                                        long long xs, signed char* __restrict__ codes, long long pitch,
                                                        unsigned char* __restrict__ scales) {
  constexpr int VEC = traits<T>::VEC, LPG = rv::GROUP / VEC;
  const int t = threadIdx.x & (tpr - 1), rg = threadIdx.x / tpr, rpb = 256 / tpr;
  const int G = (C + rv::GROUP - 1) / rv::GROUP;
  for (long long row = (long long)blockIdx.x * rpb + rg; row < rows; row += (long long)gridDim.x * rpb) {
    for (int c = t * VEC; c < G * rv::GROUP; c += tpr * VEC) {      // whole groups: every lane of one takes part
      const int at = C >= VEC ? min(c, C - VEC) : 0, skip = C >= VEC ? min(c - at, VEC) : (c ? VEC : 0);
      float v[VEC];
      load_any<T>(x + row * xs, at, C, v);
      unsigned big = 0, wd[VEC / 4];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {                               // as integers: NaN is the largest
        const unsigned a = __float_as_uint(v[i]) & 0x7fffffffu;
        big = max(big, i >= skip ? a : 0u);
      }
      const unsigned sc = rv::group_scale(rv::lanes_max<LPG>(big));
      rv::group_codes<VEC>(v, sc, wd);
      if (c < C) rv::store_codes(codes + row * pitch + c, skip, wd);
      if ((c & (rv::GROUP - 1)) == 0) scales[row * G + c / rv::GROUP] = (unsigned char)sc;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void act8_unpack_kernel(long long rows, int C, int tpr, const signed char* __restrict__ codes,
                                                          long long pitch, const unsigned char* __restrict__ scales,
                                                          T* __restrict__ y, long long ys, int ycols) {
  constexpr int VEC = traits<T>::VEC;
  const int t = threadIdx.x & (tpr - 1), rg = threadIdx.x / tpr, rpb = 256 / tpr;
  const int G = (C + rv::GROUP - 1) / rv::GROUP;
  for (long long row = (long long)blockIdx.x * rpb + rg; row < rows; row += (long long)gridDim.x * rpb) {
    for (int c = t * VEC; c < C; c += tpr * VEC) {
      const int at = C >= VEC ? min(c, C - VEC) : 0, skip = c - at;
      unsigned wd[VEC / 4];
      rv::load_codes(codes + row * pitch + at, wd);
      const float s1 = rv::group_step(scales[row * G + c / rv::GROUP]), s0 = rv::group_step(scales[row * G + at / rv::GROUP]);
      float v[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = rv::code_at(wd, i) * (i < skip ? s0 : s1);
      if (C >= VEC) {
        rv::store_vec<T>(y + row * ys + at, v);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (i < C) traits<T>::store1(y + row * ys + i, v[i]);
      }
    }
    if (ycols > C)
      for (int c = C + t; c < ycols; c += tpr) traits<T>::store1(y + row * ys + c, 0.f);
  }
}

// ------------------------------------------------------------------------------------------------ weight gradient
// dW[m][n] = sum over rows r of dY[r][m] X[r][n].  Rows are the contraction and both operands hold them as their slow
// dimension; a matrix instruction wants eight of them per lane.  A step of 32 rows is staged in LDS as it lies in memory (X
// converted to bf16 on the way) and read back with ds_read_b64_tr_b16, which hands a group of 16 lanes a 4 x 16 block
// transposed.  Row strides of 64 bytes times an odd number keep the four rows of such a block in different banks.
// A workgroup owns a (32 MB WM) x (32 NB WN) tile of dW and steps s, s + S, ...: WM WN waves share a step's staging (a
// barrier per step), or, with WM = WN = 1, each of the four waves stages its own steps.  S partial tiles go to the
// workspace, summed in a fixed order by rowvec.h's fold (S = 1: straight to dW).
constexpr int WG_ROWS = 32;

__device__ __forceinline__ bf16x8 tr_frag(const unsigned short* base, int stride, int lane) {
  // lane l of a 16-lane group reads 8 bytes of row (l & 15) >> 2, columns 4 (l & 3) ..; it receives column l & 15, four rows
  const int g = lane >> 4;                                       // groups: (columns 0-15 | 16-31) x (rows 0-7 | 8-15)
  const unsigned short* p = base + ((g >> 1) * 8 + ((lane & 15) >> 2)) * stride + (g & 1) * 16 + (lane & 3) * 4;
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4* lp;
  const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
  const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * stride));
  typedef short s8 __attribute__((ext_vector_type(8)));
  const s8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8, v);
}

constexpr int odd64(int cols) {                                  // row stride in elements: 32 times an odd number
  return ((cols / 32) & 1) ? cols : cols + 32;
}

template <int MB, int NB, int WM, int WN>
__global__ __launch_bounds__(256) void act8_wgrad_kernel(long long rows, int M, int N, const bf16* __restrict__ dY,
                                                         long long dys, const signed char* __restrict__ codes,
                                                         long long pitch, const unsigned char* __restrict__ scales,
                                                         float* __restrict__ out, int S, int tiles_n) {
  constexpr bool SHARED = WM * WN == 4;                          // four waves share the staged step
  static_assert(SHARED || (WM == 1 && WN == 1), "either the waves tile the output or each has steps of its own");
  constexpr int TM = 32 * MB * WM, TN = 32 * NB * WN;
  constexpr int LA = odd64(TM), LB = odd64(TN);
  constexpr int STEP = WG_ROWS * (LA + LB);                      // elements of one staged step
  constexpr int NT = SHARED ? 256 : 64;                          // threads that stage a step
  constexpr int QA = WG_ROWS * TM / 8 / NT, QB = (WG_ROWS * TN / 16 + NT - 1) / NT;
  constexpr int BUFS = SHARED ? 2 : 4;
  constexpr int FOLD = SHARED ? 0 : TM * TN * 2;                 // the four waves' tiles are added in LDS at the end
  __shared__ __attribute__((aligned(16))) unsigned short lds[(BUFS * STEP > FOLD ? BUFS * STEP : FOLD)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tid = SHARED ? threadIdx.x : lane;
  const int tile = blockIdx.x / S, split = blockIdx.x - tile * S;
  const int m0 = (tile / tiles_n) * TM, n0 = (tile - (tile / tiles_n) * tiles_n) * TN;
  const int G = (N + rv::GROUP - 1) / rv::GROUP;
  const long long steps = (rows + WG_ROWS - 1) / WG_ROWS;
  const long long first = SHARED ? split : (long long)split * 4 + wave, stride = SHARED ? S : (long long)S * 4;
  const int wm = SHARED ? (wave % WM) * 32 * MB : 0, wn = SHARED ? (wave / WM) * 32 * NB : 0;
  f32x16 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  rv::u4_any ra[QA];
  uint4 rb[QB];
  unsigned rs[QB];
  auto fetch = [&](long long step) {
#pragma unroll
    for (int i = 0; i < QA; ++i) {
      const int q = i * NT + tid, r = q / (TM / 8), c = m0 + (q - r * (TM / 8)) * 8;
      const long long row = step * WG_ROWS + r;
      ra[i] = rv::u4_any{0, 0, 0, 0};
      if (row < rows && c < M) {
        const bf16* p = dY + row * dys + c;
        if (c + 8 <= M) {
          ra[i] = *reinterpret_cast<const rv::u4_any*>(p);
        } else {                                                 // the last columns of a row, never past its end
          unsigned h[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] = c + e < M ? p[e].u : 0u;
          ra[i] = rv::u4_any{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
        }
      }
    }
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int q = i * NT + tid, r = q / (TN / 16), c = n0 + (q - r * (TN / 16)) * 16;
      const long long row = step * WG_ROWS + r;
      const bool in = row < rows && c < N && r < WG_ROWS;
      rb[i] = make_uint4(0, 0, 0, 0);
      rs[i] = 1;
      if (in) {                                                  // (the pitch is a multiple of 16: whole chunks)
        rb[i] = *reinterpret_cast<const uint4*>(codes + row * pitch + c);
        rs[i] = scales[row * G + c / rv::GROUP];
      }
    }
  };
  auto stage = [&](unsigned short* to) {
#pragma unroll
    for (int i = 0; i < QA; ++i) {
      const int q = i * NT + tid, r = q / (TM / 8), c = (q - r * (TM / 8)) * 8;
      *reinterpret_cast<uint4*>(to + r * LA + c) = make_uint4(ra[i].x, ra[i].y, ra[i].z, ra[i].w);
    }
    unsigned short* const tb = to + WG_ROWS * LA;
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int q = i * NT + tid, r = q / (TN / 16), c = (q - r * (TN / 16)) * 16;
      if (WG_ROWS * TN / 16 % NT == 0 || r < WG_ROWS) {
        const float step = rv::group_step(rs[i]);
        const unsigned wd[4] = {rb[i].x, rb[i].y, rb[i].z, rb[i].w};
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = rv::code_at(wd, e) * step;
        typedef traits<bf16> tb16;
        *reinterpret_cast<uint4*>(tb + r * LB + c) =
            make_uint4(tb16::p2(v[0], v[1]), tb16::p2(v[2], v[3]), tb16::p2(v[4], v[5]), tb16::p2(v[6], v[7]));
        *reinterpret_cast<uint4*>(tb + r * LB + c + 8) =
            make_uint4(tb16::p2(v[8], v[9]), tb16::p2(v[10], v[11]), tb16::p2(v[12], v[13]), tb16::p2(v[14], v[15]));
      }
    }
  };
  auto multiply = [&](const unsigned short* from) {
#pragma unroll
    for (int ks = 0; ks < WG_ROWS; ks += 16) {
      bf16x8 b[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) b[j] = tr_frag(from + WG_ROWS * LA + ks * LB + wn + j * 32, LB, lane);
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const bf16x8 a = tr_frag(from + ks * LA + wm + i * 32, LA, lane);
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], acc[i][j], 0, 0, 0);
      }
    }
  };

  if (SHARED) {
    // every thread of the workgroup runs the same number of steps
    int at = 0;
    if (first < steps) fetch(first);
    for (long long s = first; s < steps; s += stride, at ^= 1) {
      stage(lds + at * STEP);
      __syncthreads();
      if (s + stride < steps) fetch(s + stride);
      multiply(lds + at * STEP);      // the other buffer is written next; this one again after the barrier that follows
    }
  } else {
    unsigned short* const mine = lds + wave * STEP;
    if (first < steps) fetch(first);
    for (long long s = first; s < steps; s += stride) {
      stage(mine);
      if (s + stride < steps) fetch(s + stride);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");     // a wave's own LDS writes and reads: in order
      __builtin_amdgcn_wave_barrier();
      multiply(mine);
      __builtin_amdgcn_wave_barrier();
    }
  }

  // C/D layout of the 32x32 product: column = lane & 31, row = (reg & 3) + 8 (reg >> 2) + 4 (lane >> 5)
  float* const dst = out + (S > 1 ? (size_t)split * M * N : 0);
  if (SHARED) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int n = n0 + wn + j * 32 + (lane & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int m = m0 + wm + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
          if (m < M && n < N) dst[(size_t)m * N + n] = acc[i][j][r];
        }
      }
  } else {
    float* const fold = reinterpret_cast<float*>(lds);
    for (int w = 0; w < 4; ++w) {
      __syncthreads();
      if (wave == w) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int at = (i * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * TN + j * 32 + (lane & 31);
              fold[at] = w ? fold[at] + acc[i][j][r] : acc[i][j][r];
            }
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < TM * TN; e += 256) {
      const int m = m0 + e / TN, n = n0 + e % TN;
      if (m < M && n < N) dst[(size_t)m * N + n] = fold[e];
    }
  }
}

// tile and number of row splits of a call
struct wg_plan { int kind, tm, tn, S; };

wg_plan wgrad_plan(long long rows, int M, int N) {
  wg_plan p;
  if (M > 64 && N > 64) { p.kind = 0; p.tm = 128; p.tn = 128; }
  else if (M > 32 && N > 32) { p.kind = 1; p.tm = 64; p.tn = 64; }
  else if (M > 32) { p.kind = 2; p.tm = 64; p.tn = 32; }
  else if (N > 32) { p.kind = 3; p.tm = 32; p.tn = 64; }
  else { p.kind = 4; p.tm = 32; p.tn = 32; }
  const long long tiles = (long long)pvn3d_ceil_div(M, p.tm) * pvn3d_ceil_div(N, p.tn);
  const long long steps = (rows + WG_ROWS - 1) / WG_ROWS;
  const long long per = p.kind == 0 ? 4 : 16;                    // steps a workgroup should have at least
  long long S = 768 / tiles;
  if (S > (steps + per - 1) / per) S = (steps + per - 1) / per;
  p.S = (int)(S < 1 ? 1 : S);
  return p;
}

#define A8_ST ((hipStream_t)stream)

int pack_threads(int C, int vec) {
  int t = 32 / vec;                                              // a whole group at least
  while (t < 64 && t * vec < C) t <<= 1;
  return t;
}
unsigned row_grid(long long rows, int tpr) {
  const long long n = (rows + 256 / tpr - 1) / (256 / tpr);
  return (unsigned)(n < 8192 ? n : 8192);
}

template <typename T>
int run_pack(long long rows, int C, const void* x, long long xs, void* codes, long long pitch, void* scales, hipStream_t st) {
  const int tpr = pack_threads(C, traits<T>::VEC);
  hipLaunchKernelGGL((act8_pack_kernel<T>), dim3(row_grid(rows, tpr)), dim3(256), 0, st, rows, C, tpr, (const T*)x, xs,
                     (signed char*)codes, pitch, (unsigned char*)scales);
  PVN3D_LAUNCH_CHECK();
  return 0;
}
template <typename T>
int run_unpack(long long rows, int C, const void* codes, long long pitch, const void* scales, void* y, long long ys, int ycols,
               hipStream_t st) {
  const int tpr = pack_threads(ycols, traits<T>::VEC);
  hipLaunchKernelGGL((act8_unpack_kernel<T>), dim3(row_grid(rows, tpr)), dim3(256), 0, st, rows, C, tpr,
                     (const signed char*)codes, pitch, (const unsigned char*)scales, (T*)y, ys, ycols);
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int pvn3d_act8_pack(int dtype, long long rows, int C, const void* x, long long xs, void* codes, long long pitch,
                               void* scales, void* stream) {
  if (dtype < 0 || dtype > 2 || C <= 0 || xs < 0 || (pitch & 15) || pitch < C) return (int)hipErrorInvalidValue;
  if (rows <= 0) return 0;
  if (!x || !codes || !scales) return (int)hipErrorInvalidValue;
  switch (dtype) {
    case 0: return run_pack<float>(rows, C, x, xs, codes, pitch, scales, A8_ST);
    case 1: return run_pack<bf16>(rows, C, x, xs, codes, pitch, scales, A8_ST);
    default: return run_pack<fp16>(rows, C, x, xs, codes, pitch, scales, A8_ST);
  }
}

extern "C" int pvn3d_act8_unpack(int dtype, long long rows, int C, const void* codes, long long pitch, const void* scales,
                                 void* y, long long ys, int y_cols, void* stream) {
  if (dtype < 0 || dtype > 2 || C <= 0 || (pitch & 15) || pitch < C || y_cols < C || ys < y_cols)
    return (int)hipErrorInvalidValue;
  if (rows <= 0) return 0;
  if (!codes || !scales || !y) return (int)hipErrorInvalidValue;
  switch (dtype) {
    case 0: return run_unpack<float>(rows, C, codes, pitch, scales, y, ys, y_cols, A8_ST);
    case 1: return run_unpack<bf16>(rows, C, codes, pitch, scales, y, ys, y_cols, A8_ST);
    default: return run_unpack<fp16>(rows, C, codes, pitch, scales, y, ys, y_cols, A8_ST);
  }
}

extern "C" size_t pvn3d_act8_wgrad_workspace_bytes(long long rows, int M, int N) {
  if (rows <= 0 || M <= 0 || N <= 0) return 0;
  const wg_plan p = wgrad_plan(rows, M, N);
  return p.S > 1 ? (size_t)p.S * M * N * sizeof(float) : 0;
}

extern "C" int pvn3d_act8_wgrad(long long rows, int M, int N, const void* dY, long long dys, const void* codes,
                                long long pitch, const void* scales, float* dW, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (M < 0 || N < 0 || dys < 0 || (pitch & 15) || pitch < N) return (int)hipErrorInvalidValue;
  if (M == 0 || N == 0) return 0;
  if (!dW) return (int)hipErrorInvalidValue;
  if (rows <= 0) {
    pvn3d_fill_u32(dW, 0, (size_t)M * N, A8_ST);
    PVN3D_LAUNCH_CHECK();
    return 0;
  }
  if (!dY || !codes || !scales) return (int)hipErrorInvalidValue;
  const wg_plan p = wgrad_plan(rows, M, N);
  const size_t count = (size_t)M * N;
  if (p.S > 1 && (!workspace || workspace_bytes < p.S * count * sizeof(float))) return (int)hipErrorInvalidValue;
  float* const out = p.S > 1 ? (float*)workspace : dW;
  const int tn = pvn3d_ceil_div(N, p.tn);
  const long long blocks = (long long)pvn3d_ceil_div(M, p.tm) * tn * p.S;
  if (blocks > 0x7fffffffLL) return (int)hipErrorInvalidValue;
#define A8_CALL(MB, NB, WM, WN)                                                                                      \
  hipLaunchKernelGGL((act8_wgrad_kernel<MB, NB, WM, WN>), dim3((unsigned)blocks), dim3(256), 0, A8_ST, rows, M, N,  \
                     (const bf16*)dY, dys, (const signed char*)codes, pitch, (const unsigned char*)scales, out, p.S, tn)
  switch (p.kind) {
    case 0: A8_CALL(2, 2, 2, 2); break;
    case 1: A8_CALL(2, 2, 1, 1); break;
    case 2: A8_CALL(2, 1, 1, 1); break;
    case 3: A8_CALL(1, 2, 1, 1); break;
    default: A8_CALL(1, 1, 1, 1); break;
  }
#undef A8_CALL
  PVN3D_LAUNCH_CHECK();
  return p.S > 1 ? rv::fold(p.S, count, count, (const float*)workspace, dW, nullptr, A8_ST) : 0;
}
