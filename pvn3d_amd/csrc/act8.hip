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
// tpr threads across a row (a power of two that covers the row, or whole groups of it), 256 / tpr rows a pass and two passes
// in flight.  Chunks are windows (rowvec.h), addresses a base the workgroup shares plus a 32-bit offset; a row shorter than a
// chunk is read value by value.  LPG: lanes per group, fewer than a whole group's if the row is shorter.
// Bound by HBM: bf16 786432 x 96 packed in 38 us (6.0 TB/s), unpacked in 34 us (6.8 TB/s, partly from the cache behind L2).
constexpr int FLY = 2;

template <typename T, int LPG>
__global__ __launch_bounds__(256) void act8_pack_kernel(long long rows, int C, int tpr, const T* __restrict__ x, int xs,
                                                        signed char* __restrict__ codes, int pitch,
                                                        unsigned char* __restrict__ scales) {
  constexpr int VEC = traits<T>::VEC;
  const int t = threadIdx.x & (tpr - 1), rg = threadIdx.x / tpr, rpb = 256 / tpr;
  const int G = (C + rv::GROUP - 1) / rv::GROUP, across = (C + LPG * VEC - 1) / (LPG * VEC) * (LPG * VEC);
  for (long long base = (long long)blockIdx.x * rpb * FLY; base < rows; base += (long long)gridDim.x * rpb * FLY) {
    const int last = (int)(rows - 1 - base < rpb * FLY - 1 ? rows - 1 - base : rpb * FLY - 1);
    const T* const xb = x + base * xs;
    signed char* const cb = codes + base * pitch;
    unsigned char* const sb = scales + base * G;
    for (int c = t * VEC; c < across; c += tpr * VEC) {             // whole groups: every lane of one takes part
      const int at = C >= VEC ? min(c, C - VEC) : 0, skip = C >= VEC ? min(c - at, VEC) : (c ? VEC : 0);
      rv::u4_any raw[FLY];
#pragma unroll
      for (int r = 0; r < FLY; ++r) {
        const T* const p = rv::at32(xb, (__umul24(min(rg + r * rpb, last), xs) + at) * (unsigned)sizeof(T));
        if (C >= VEC) {
          raw[r] = *reinterpret_cast<const rv::u4_any*>(p);
        } else {
          float v[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[i] = i < C ? traits<T>::load1(p + i) : 0.f;
          raw[r] = traits<T>::pack(v);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < FLY; ++r) {
        const int rl = rg + r * rpb;
        float v[VEC];
        traits<T>::unpack(raw[r], v);
        unsigned big = 0, wd[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {                             // as integers: NaN is the largest
          const unsigned a = __float_as_uint(v[i]) & 0x7fffffffu;
          big = max(big, i >= skip ? a : 0u);
        }
        const unsigned sc = rv::group_scale(rv::lanes_max<LPG>(big));
        rv::group_codes<VEC>(v, sc, wd);
        if (rl <= last && c < C) {
          rv::store_codes(rv::at32(cb, __umul24(rl, pitch) + c), skip, wd);
          if ((c & (rv::GROUP - 1)) == 0) *rv::at32(sb, __umul24(rl, G) + c / rv::GROUP) = (unsigned char)sc;
        }
      }
    }
  }
}

template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void act8_unpack_kernel(long long rows, int C, int tpr,
                                                          const signed char* __restrict__ codes, int pitch,
                                                          const unsigned char* __restrict__ scales, T* __restrict__ y, int ys,
                                                          int ycols) {
  constexpr int VEC = traits<T>::VEC;
  const int t = threadIdx.x & (tpr - 1), rg = threadIdx.x / tpr, rpb = 256 / tpr;
  const int G = (C + rv::GROUP - 1) / rv::GROUP;
  for (long long base = (long long)blockIdx.x * rpb * FLY; base < rows; base += (long long)gridDim.x * rpb * FLY) {
    const int last = (int)(rows - 1 - base < rpb * FLY - 1 ? rows - 1 - base : rpb * FLY - 1);
    const signed char* const cb = codes + base * pitch;
    const unsigned char* const sb = scales + base * G;
    T* const yb = y + base * ys;
    for (int c = t * VEC; c < C; c += tpr * VEC) {
      const int at = C >= VEC ? min(c, C - VEC) : 0, skip = c - at;
      unsigned wd[FLY][VEC / 4];
      unsigned char s0[FLY], s1[FLY];
#pragma unroll
      for (int r = 0; r < FLY; ++r) {
        const int rl = min(rg + r * rpb, last);
        rv::load_codes(rv::at32(cb, __umul24(rl, pitch) + at), wd[r]);
        s1[r] = *rv::at32(sb, __umul24(rl, G) + c / rv::GROUP);
        s0[r] = *rv::at32(sb, __umul24(rl, G) + at / rv::GROUP);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < FLY; ++r) {
        const int rl = rg + r * rpb;
        const float f1 = rv::group_step(s1[r]), f0 = rv::group_step(s0[r]);
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = rv::code_at(wd[r], i) * (i < skip ? f0 : f1);
        if (rl <= last) {
          T* const p = rv::at32(yb, (__umul24(rl, ys) + at) * (unsigned)sizeof(T));
          if (C >= VEC) {
            rv::store_vec<T, STREAM>(p, v);
          } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              if (i < C) traits<T>::store1(p + i, v[i]);
          }
        }
      }
    }
    if (ycols > C) {
      for (int rl = rg; rl <= last; rl += rpb)
#pragma unroll 1
        for (int c = C + t; c < ycols; c += tpr)
          traits<T>::store1(rv::at32(yb, (__umul24(rl, ys) + c) * (unsigned)sizeof(T)), 0.f);
    }
  }
}

// ------------------------------------------------------------------------------------------------ weight gradient
// dW[m][n] = sum over rows r of dY[r][m] X[r][n].  Rows are the contraction and both operands hold them as their slow
// dimension; a matrix instruction wants eight of them per lane.  A step of 32 or 64 rows is staged in LDS as it lies in memory
// (X converted to bf16 on the way) and read back with ds_read_b64_tr_b16, which hands a group of 16 lanes a 4 x 16 block
// transposed.  Row strides of 64 bytes times an odd number keep the four rows of such a block in different banks.
// A workgroup owns a (32 MB WM) x (32 NB WN) tile of dW and steps s, s + S, ... of ROWS rows: WM WN waves share a step's
// staging (a barrier per step), or, with WM = WN = 1, each of four waves stages its own steps.  S partial tiles go to the
// workspace, summed in a fixed order by rowvec.h's fold (S = 1: straight to dW).
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

// What bounds it: HBM for narrow layers (1572864 rows, 64 x 32: 45 us with the sum of 512 partial tiles, 5.6 TB/s).
// For wide ones how much the two waves of a SIMD overlap: a step of 64 rows of the 256 x 128 tile keeps the matrix pipes busy
// for 45 % of its cycles, LDS (176 KB) for 45 %, the vector units for 22 %.  12288 rows, 512 x 1536 take 33.6 us with the sum
// of the 31.5 MB of partial tiles, 575 TFLOP/s; 98304 rows, 512 x 512 78 us, 661 TFLOP/s (the library's bf16 product: 81 and
// 311 us; its rate for a large square one: 1257 TFLOP/s).
constexpr int odd64(int cols) {                                  // row stride in elements: 32 times an odd number
  return ((cols / 32) & 1) ? cols : cols + 32;
}

// 8 values that start `skip` places late, moved down (the places freed get zeros)
__device__ __forceinline__ uint4 shift_down(const rv::u4_any& v, int skip) {
  const unsigned long long lo = ((unsigned long long)v.y << 32) | v.x, hi = ((unsigned long long)v.w << 32) | v.z;
  const int b = 16 * (skip & 3);
  unsigned long long l = b ? (lo >> b) | (hi << (64 - b)) : lo, h = hi >> b;
  if (skip & 4) { l = h; h = 0; }
  return make_uint4((unsigned)l, (unsigned)(l >> 32), (unsigned)h, (unsigned)(h >> 32));
}

// Every load is whole and unconditional -- rows behind the last repeat it (their dY is zeroed and their scale set to 1 when
// they are staged), columns behind the last repeat others and end in columns of the tile that are not stored -- and its
// address is a base the workgroup shares plus a 32-bit offset.  RAGGED: M is no multiple of 8.
template <int MB, int NB, int WM, int WN, int ROWS, bool RAGGED, bool STREAM>
__global__ __launch_bounds__(WM * WN > 1 ? 64 * WM * WN : 256) void act8_wgrad_kernel(
    long long rows, int M, int N, const bf16* __restrict__ dY, int dys, const signed char* __restrict__ codes, int pitch,
    const unsigned char* __restrict__ scales, float* __restrict__ out, int S, int tiles_n) {
  constexpr bool SHARED = WM * WN > 1;                           // the waves share the staged step
  static_assert(SHARED || ROWS == 32, "a wave on its own takes 32 rows a step");
  constexpr int TM = 32 * MB * WM, TN = 32 * NB * WN;
  constexpr int LA = odd64(TM), LB = odd64(TN);
  constexpr int STEP = ROWS * (LA + LB);                      // elements of one staged step
  constexpr int NT = 64 * WM * WN;                              // threads that stage a step
  constexpr int QA = ROWS * TM / 8 / NT, QB = ROWS * TN / 16 / NT;
  static_assert(QA >= 1 && QB >= 1, "every thread has a chunk of both");
  constexpr int BUFS = SHARED ? 2 : 4;
  constexpr int FOLD = SHARED ? 0 : TM * TN * 2;                 // the four waves' tiles are added in LDS at the end
  __shared__ __attribute__((aligned(16))) unsigned short lds[(BUFS * STEP > FOLD ? BUFS * STEP : FOLD)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tid = SHARED ? threadIdx.x : lane;
  const int tile = blockIdx.x / S, split = blockIdx.x - tile * S;
  const int m0 = (tile / tiles_n) * TM, n0 = (tile - (tile / tiles_n) * tiles_n) * TN;
  const int G = (N + rv::GROUP - 1) / rv::GROUP;
  const int whole = (int)(rows / ROWS), rest = (int)(rows - (long long)whole * ROWS);
  const int first = SHARED ? split : __builtin_amdgcn_readfirstlane(split * 4 + wave), stride = SHARED ? S : S * 4;
  const int wm = SHARED ? (wave % WM) * 32 * MB : 0, wn = SHARED ? (wave / WM) * 32 * NB : 0;
  f32x16 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // this thread's chunks: row of the step, column (in memory: the window that holds it)
  int ar[QA], ac[QA], askip[QA], br[QB], bc[QB];
#pragma unroll
  for (int i = 0; i < QA; ++i) {
    const int q = i * NT + tid, c = m0 + q % (TM / 8) * 8;
    ar[i] = q / (TM / 8);
    ac[i] = min(c, max(M - 8, 0));
    askip[i] = min(c - ac[i], 8);
  }
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int q = i * NT + tid;
    br[i] = q / (TN / 16);
    bc[i] = min(n0 + q % (TN / 16) * 16, (N - 1) & ~15);         // (the pitch is a multiple of 16: whole chunks)
  }
  struct held {
    rv::u4_any a[QA];
    uint4 b[QB];
    unsigned char s[QB];
  };
  // last_step: the step of the rows behind the last whole one
  auto fetch = [&](int step, held& h, bool last_step) {
    const bf16* const pa = dY + (long long)step * ROWS * dys;
    const signed char* const pb = codes + (long long)step * ROWS * pitch;
    const unsigned char* const ps = scales + (long long)step * ROWS * G;
#pragma unroll
    for (int i = 0; i < QA; ++i) {
      const bf16* const p = rv::at32(pa, (__umul24(last_step ? min(ar[i], rest - 1) : ar[i], dys) + ac[i]) * 2u);
      if (RAGGED && M < 8) {                                     // rows shorter than a chunk: value by value
        unsigned v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p[min(e, M - 1)].u;
        h.a[i] = rv::u4_any{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
      } else {
        rv::get<STREAM>(p, h.a[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int r = last_step ? min(br[i], rest - 1) : br[i];
      rv::u4_any b;
      rv::get<STREAM>(rv::at32(pb, __umul24(r, pitch) + bc[i]), b);
      h.b[i] = make_uint4(b.x, b.y, b.z, b.w);
      h.s[i] = *rv::at32(ps, __umul24(r, G) + bc[i] / rv::GROUP);
    }
  };
  auto stage = [&](unsigned short* to, const held& h, bool last_step) {
#pragma unroll
    for (int i = 0; i < QA; ++i) {
      uint4 v = make_uint4(h.a[i].x, h.a[i].y, h.a[i].z, h.a[i].w);
      if (RAGGED && M >= 8) v = shift_down(h.a[i], askip[i]);
      if (last_step && ar[i] >= rest) v = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(to + ar[i] * LA + (i * NT + tid) % (TM / 8) * 8) = v;
    }
    unsigned short* const tb = to + ROWS * LA;
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const float two = rv::group_step(last_step && br[i] >= rest ? 1u : h.s[i]);
      const unsigned wd[4] = {h.b[i].x, h.b[i].y, h.b[i].z, h.b[i].w};
      unsigned v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = traits<bf16>::p2(rv::code_at(wd, 2 * e) * two, rv::code_at(wd, 2 * e + 1) * two);
      uint4* const p = reinterpret_cast<uint4*>(tb + br[i] * LB + (i * NT + tid) % (TN / 16) * 16);
      p[0] = make_uint4(v[0], v[1], v[2], v[3]);
      p[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
  };
  constexpr int KS = 2;
  struct frags { bf16x8 a[KS][MB], b[KS][NB]; };
  auto read = [&](const unsigned short* from, frags& f, int k0) {
#pragma unroll
    for (int k = 0; k < KS; ++k) {
#pragma unroll
      for (int j = 0; j < NB; ++j) f.b[k][j] = tr_frag(from + ROWS * LA + (k0 + k * 16) * LB + wn + j * 32, LB, lane);
#pragma unroll
      for (int i = 0; i < MB; ++i) f.a[k][i] = tr_frag(from + (k0 + k * 16) * LA + wm + i * 32, LA, lane);
    }
  };
  auto multiply = [&](const frags& f) {
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.a[k][i], f.b[k][j], acc[i][j], 0, 0, 0);
  };

  const int n = first < whole ? (whole - 1 - first) / stride + 1 : 0;          // whole steps of this workgroup (wave)
  held h;
  if (SHARED) {
    // One barrier a step: behind it the step's fragments are read, the next step (in registers since the last barrier) is
    // converted into the other buffer -- which every wave has read before it came to this barrier -- and the products run
    // beside that.  What is fetched and staged ahead of the last step is never multiplied.
    if (n > 0) {
      auto step_at = [&](int i) { return first + min(i, n - 1) * stride; };
      fetch(step_at(0), h, false);
      stage(lds, h, false);
      fetch(step_at(1), h, false);
      for (int i = 0; i < n; i += 2) {
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          if (i + d < n) {           // (the same for the whole workgroup)
            frags f;
            __syncthreads();
            read(lds + (d & 1) * STEP, f, 0);
            stage(lds + ((d & 1) ^ 1) * STEP, h, false);
            fetch(step_at(i + d + 2), h, false);
            multiply(f);
#pragma unroll
            for (int k = 32; k < ROWS; k += 32) {
              read(lds + (d & 1) * STEP, f, k);
              multiply(f);
            }
          }
        }
      }
    }
    if (rest && whole % S == split) {                            // the rows behind the last whole step
      frags f;
      __syncthreads();
      fetch(whole, h, true);
      stage(lds, h, true);
      __syncthreads();
      for (int k = 0; k < ROWS; k += 32) {
        read(lds, f, k);
        multiply(f);
      }
    }
  } else {
    unsigned short* const mine = lds + wave * STEP;
    if (n > 0) fetch(first, h, false);
    for (int i = 0; i < n; ++i) {
      frags f;
      stage(mine, h, false);
      fetch(first + min(i + 1, n - 1) * stride, h, false);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");     // a wave's own LDS writes and reads: in order
      __builtin_amdgcn_wave_barrier();
      read(mine, f, 0);
      multiply(f);
      __builtin_amdgcn_wave_barrier();
    }
    if (rest && whole % (S * 4) == first) {
      frags f;
      fetch(whole, h, true);
      stage(mine, h, true);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      read(mine, f, 0);
      multiply(f);
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

// Tile, rows of a step and number of row splits of a call.  Every split leaves a partial tile that is written and read
// again, so there are no more workgroups than keep the chip busy: one of eight waves per CU for the 256 x 128 tile (33.5 MB of
// partial sums at most; 98304 x 512 x 512: 78 us, 87 us with two per CU), two of four waves for the others (786432 x 96 x 64:
// 43 us, 55 with one, 54 with three; 1572864 x 32 x 16: 27, 37, 28).  The 256 x 128 tile converts each code for twice the
// output; up to 128 output channels half of it would be empty (393216 x 128 x 128: 128 x 128).
struct wg_plan { int kind, tm, tn, S; };

wg_plan wgrad_plan(long long rows, int M, int N) {
  wg_plan p;
  int step = 32, wgs = 512, per = 16;                            // per: steps a workgroup should have at least
  if (M > 128 && N > 64) { p.kind = 0; p.tm = 256; p.tn = 128; step = 64; wgs = 256; per = 4; }
  else if (M > 64 && N > 64) { p.kind = 1; p.tm = 128; p.tn = 128; step = 64; per = 4; }
  else if (M > 32 && N > 64) { p.kind = 2; p.tm = 64; p.tn = 128; step = 64; per = 4; }
  else if (M > 64 && N > 32) { p.kind = 3; p.tm = 128; p.tn = 64; step = 64; per = 4; }
  else if (M > 32 && N > 32) { p.kind = 4; p.tm = 64; p.tn = 64; }
  else if (M > 32) { p.kind = 5; p.tm = 64; p.tn = 32; }
  else if (N > 32) { p.kind = 6; p.tm = 32; p.tn = 64; }
  else { p.kind = 7; p.tm = 32; p.tn = 32; }
  const long long tiles = (long long)pvn3d_ceil_div(M, p.tm) * pvn3d_ceil_div(N, p.tn);
  const long long steps = (rows + step - 1) / step;
  long long S = wgs / tiles;
  if (S > (steps + per - 1) / per) S = (steps + per - 1) / per;
  // Workgroup numbers are tile S + split and are dealt to the eight XCDs in turn: with a multiple of eight the tiles of a split
  // are on one XCD and find its rows in that one's L2 (400000 x 20 x 130: 24.8 us, 39.0 with 170 splits; 200000 x 200 x 300: 60,
  // 64).  Below 32 splits too many CUs would go without work (98304 x 520 x 260: 85 us with 24 splits, 75 with 28).
  if (S >= 32) S = S / 8 * 8;
  p.S = (int)(S < 1 ? 1 : S);
  return p;
}

// ------------------------------------------------------------------------------------------------ columns kept exact
// dW[m][k] = sum over rows of dY[r][m] X[r][k] for K <= 8 bf16 columns X: inputs that are no layer's outputs (a neighbour's
// relative coordinates, colours, normals) and would lose their bits to the larger channels of a group of 32 are kept beside
// the codes as they are.  A thread owns 8 columns of dY and all of X's; across (a power of two, 32 at most) threads share a
// row, 256 / across rows a pass, two passes in flight.  Exact products, fp32 sums in a fixed order, partial sums as above.
// Bound by HBM (dY is read once) and, narrow, by its two launches: 786432 x 64, 3 columns 24 us (4.3 TB/s), 98304 x 256 17 us.
template <int KM>
__global__ __launch_bounds__(256) void act8_columns_kernel(long long rows, int M, int K, int across,
                                                           const bf16* __restrict__ dY, int dys, const bf16* __restrict__ X,
                                                           int xs, float* __restrict__ out) {
  constexpr int VEC = 8;
  __shared__ float red[256 * VEC];
  const int t = threadIdx.x & (across - 1), slot = threadIdx.x / across, slots = 256 / across;
  const int c = ((int)blockIdx.y * across + t) * VEC;
  const int at = M >= VEC ? min(c, M - VEC) : 0;                               // (M < 8: read value by value)
  float acc[VEC][KM];
#pragma unroll
  for (int i = 0; i < VEC; ++i)
#pragma unroll
    for (int k = 0; k < KM; ++k) acc[i][k] = 0.f;
  for (long long base = (long long)blockIdx.x * slots * FLY; base < rows; base += (long long)gridDim.x * slots * FLY) {
    const int last = (int)(rows - 1 - base < slots * FLY - 1 ? rows - 1 - base : slots * FLY - 1);
    const bf16* const db = dY + base * dys;
    const bf16* const xb = X + base * xs;
    rv::u4_any raw[FLY];
    unsigned short xv[FLY][KM];
#pragma unroll
    for (int r = 0; r < FLY; ++r) {
      const int rl = min(slot + r * slots, last);
      const bf16* const p = rv::at32(db, (__umul24(rl, dys) + at) * 2u);
      if (M >= VEC) {
        raw[r] = *reinterpret_cast<const rv::u4_any*>(p);
      } else {
        unsigned v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = p[min(i, M - 1)].u;
        raw[r] = rv::u4_any{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
      }
#pragma unroll
      for (int k = 0; k < KM; ++k) xv[r][k] = rv::at32(xb, (__umul24(rl, xs) + min(k, K - 1)) * 2u)->u;
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < FLY; ++r) {
      if (slot + r * slots <= last) {
        float d[VEC];
        traits<bf16>::unpack(raw[r], d);
#pragma unroll
        for (int k = 0; k < KM; ++k) {
          const float x = __uint_as_float((unsigned)xv[r][k] << 16);
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i][k] = fmaf(d[i], x, acc[i][k]);
        }
      }
    }
  }
  // over the row slots, column by column of X
  float* const dst = out + (size_t)blockIdx.x * M * K;
#pragma unroll
  for (int k = 0; k < KM; ++k) {
    if (k < K) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VEC; ++i) red[slot * across * VEC + t * VEC + i] = acc[i][k];
      __syncthreads();
      for (int e = threadIdx.x; e < across * VEC; e += 256) {
        const int ce = ((int)blockIdx.y * across + e / VEC) * VEC, ae = M >= VEC ? min(ce, M - VEC) : 0, m = ae + e % VEC;
        if (ce < M && e % VEC >= ce - ae && m < M) {
          float s = 0.f;
          for (int q = 0; q < slots; ++q) s += red[q * across * VEC + e];
          dst[(size_t)m * K + k] = s;
        }
      }
    }
  }
}

struct columns_plan { int across, tiles, S; };

columns_plan columns_grid(long long rows, int M) {
  columns_plan p;
  const int chunks = (M + 7) / 8;
  p.across = 1;
  while (p.across < chunks && p.across < 32) p.across <<= 1;
  p.tiles = (chunks + p.across - 1) / p.across;
  const long long per = 256 / p.across * FLY, n = (rows + per - 1) / per;      // passes; a workgroup makes four or more
  long long S = 1024 / p.tiles;
  if (S > (n + 3) / 4) S = (n + 3) / 4;
  p.S = (int)(S < 1 ? 1 : S);
  return p;
}

constexpr long long MAX_STRIDE = 1 << 20;      // a workgroup's rows are within 32-bit offsets of their base
constexpr long long MAX_ROWS = 1ll << 35;      // steps are counted in 32 bits

#define A8_ST ((hipStream_t)stream)

int row_threads(int C, int vec) {                                // threads across a row
  int t = 1;
  while (t < 64 && t * vec < C) t <<= 1;
  return t;
}
unsigned row_grid(long long rows, int tpr) {
  const int per = 256 / tpr * FLY;
  // packed and unpacked: bf16 786432 x 96 77.0 us (4096: 83, 8192: 79, 24576: 80), fp32 1000000 x 33 56 (57, 56, 59)
  return rv::even_grid((rows + per - 1) / per, 12288);
}

template <typename T>
int run_pack(long long rows, int C, const void* x, long long xs, void* codes, long long pitch, void* scales, hipStream_t st) {
  const int tpr = row_threads(C, traits<T>::VEC);
#define A8_PACK(LPG)                                                                                                        \
  hipLaunchKernelGGL((act8_pack_kernel<T, LPG>), dim3(row_grid(rows, tpr)), dim3(256), 0, st, rows, C, tpr, (const T*)x,    \
                     (int)xs, (signed char*)codes, (int)pitch, (unsigned char*)scales)
  const int lpg = tpr < rv::GROUP / traits<T>::VEC ? tpr : rv::GROUP / traits<T>::VEC;
  if (lpg == 1) A8_PACK(1);
  else if (lpg == 2) A8_PACK(2);
  else if (lpg == 4) A8_PACK(4);
  else A8_PACK((traits<T>::VEC == 4 ? 8 : 4));
#undef A8_PACK
  PVN3D_LAUNCH_CHECK();
  return 0;
}
template <typename T>
int run_unpack(long long rows, int C, const void* codes, long long pitch, const void* scales, void* y, long long ys,
               int ycols, hipStream_t st) {
  const int tpr = row_threads(C, traits<T>::VEC);
#define A8_UNPACK(STREAM)                                                                                                  \
  hipLaunchKernelGGL((act8_unpack_kernel<T, STREAM>), dim3(row_grid(rows, tpr)), dim3(256), 0, st, rows, C, tpr,           \
                     (const signed char*)codes, (int)pitch, (const unsigned char*)scales, (T*)y, (int)ys, ycols)
  if (rows * C * (long long)sizeof(T) >= rv::STREAM_BYTES) A8_UNPACK(true);
  else A8_UNPACK(false);
#undef A8_UNPACK
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int pvn3d_act8_pack(int dtype, long long rows, int C, const void* x, long long xs, void* codes, long long pitch,
                               void* scales, void* stream) {
  if (dtype < 0 || dtype > 2 || C <= 0 || xs < 0 || (pitch & 15) || pitch < C || xs > MAX_STRIDE || pitch > MAX_STRIDE)
    return (int)hipErrorInvalidValue;
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
  if (dtype < 0 || dtype > 2 || C <= 0 || (pitch & 15) || pitch < C || y_cols < C || ys < y_cols || ys > MAX_STRIDE ||
      pitch > MAX_STRIDE)
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
  if (M < 0 || N < 0 || dys < 0 || (pitch & 15) || pitch < N || dys > MAX_STRIDE || pitch > MAX_STRIDE)
    return (int)hipErrorInvalidValue;
  if (M == 0 || N == 0) return 0;
  if (!dW) return (int)hipErrorInvalidValue;
  if (rows <= 0) {
    pvn3d_fill_u32(dW, 0, (size_t)M * N, A8_ST);
    PVN3D_LAUNCH_CHECK();
    return 0;
  }
  if (!dY || !codes || !scales || rows > MAX_ROWS) return (int)hipErrorInvalidValue;
  const wg_plan p = wgrad_plan(rows, M, N);
  const size_t count = (size_t)M * N;
  if (p.S > 1 && (!workspace || ((size_t)workspace & 15) || workspace_bytes < p.S * count * sizeof(float)))
    return (int)hipErrorInvalidValue;
  float* const out = p.S > 1 ? (float*)workspace : dW;
  const int tn = pvn3d_ceil_div(N, p.tn);
  const long long blocks = (long long)pvn3d_ceil_div(M, p.tm) * tn * p.S;
  if (blocks > 0x7fffffffLL) return (int)hipErrorInvalidValue;
  // a single tile reads its rows once (1572864 x 64 x 32: 45.3 us past the caches, 48.0; tiles that waves share are the slower
  // for it, 800000 x 100 x 100 60, 57)
  const bool once = p.kind >= 4 && blocks == p.S && rows * (2 * M + (long long)N) >= rv::STREAM_BYTES;
#define A8_ONE(MB, NB, WM, WN, ROWS, RAG, STREAM)                                                                           \
  hipLaunchKernelGGL((act8_wgrad_kernel<MB, NB, WM, WN, ROWS, RAG, STREAM>), dim3((unsigned)blocks),                                \
                     dim3(WM * WN > 1 ? 64 * WM * WN : 256), 0, A8_ST, rows, M, N, (const bf16*)dY, (int)dys,               \
                     (const signed char*)codes, (int)pitch, (const unsigned char*)scales, out, p.S, tn)
#define A8_CALL(MB, NB, WM, WN, ROWS)                        \
  do {                                                       \
    if (M & 7) A8_ONE(MB, NB, WM, WN, ROWS, true, false);    \
    else A8_ONE(MB, NB, WM, WN, ROWS, false, false);         \
  } while (0)
#define A8_NARROW(MB, NB)                                    \
  do {                                                       \
    if (!once) A8_CALL(MB, NB, 1, 1, 32);                    \
    else if (M & 7) A8_ONE(MB, NB, 1, 1, 32, true, true);    \
    else A8_ONE(MB, NB, 1, 1, 32, false, true);              \
  } while (0)
  switch (p.kind) {
    case 0: A8_CALL(2, 2, 4, 2, 64); break;
    case 1: A8_CALL(2, 2, 2, 2, 64); break;
    case 2: A8_CALL(1, 2, 2, 2, 64); break;
    case 3: A8_CALL(2, 1, 2, 2, 64); break;
    case 4: A8_NARROW(2, 2); break;
    case 5: A8_NARROW(2, 1); break;
    case 6: A8_NARROW(1, 2); break;
    default: A8_NARROW(1, 1); break;
  }
#undef A8_ONE
#undef A8_CALL
#undef A8_NARROW
  PVN3D_LAUNCH_CHECK();
  return p.S > 1 ? rv::fold(p.S, count, count, (const float*)workspace, dW, nullptr, A8_ST) : 0;
}

constexpr int MAX_COLUMNS = 8;

extern "C" size_t pvn3d_act8_columns_workspace_bytes(long long rows, int M, int K) {
  if (rows <= 0 || M <= 0 || K <= 0 || K > MAX_COLUMNS) return 0;
  const columns_plan p = columns_grid(rows, M);
  return p.S > 1 ? (size_t)p.S * M * K * sizeof(float) : 0;
}

extern "C" int pvn3d_act8_columns_wgrad(long long rows, int M, int K, const void* dY, long long dys, const void* X,
                                        long long xs, float* dW, void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || K < 0 || K > MAX_COLUMNS || dys < 0 || xs < 0 || dys > MAX_STRIDE || xs > MAX_STRIDE)
    return (int)hipErrorInvalidValue;
  if (M == 0 || K == 0) return 0;
  if (!dW) return (int)hipErrorInvalidValue;
  if (rows <= 0) {
    pvn3d_fill_u32(dW, 0, (size_t)M * K, A8_ST);
    PVN3D_LAUNCH_CHECK();
    return 0;
  }
  const columns_plan p = columns_grid(rows, M);
  const size_t count = (size_t)M * K;
  if (!dY || !X || p.tiles > 65535) return (int)hipErrorInvalidValue;
  if (p.S > 1 && (!workspace || ((size_t)workspace & 15) || workspace_bytes < p.S * count * sizeof(float)))
    return (int)hipErrorInvalidValue;
  float* const out = p.S > 1 ? (float*)workspace : dW;
#define A8_COLUMNS(KM)                                                                                                      \
  hipLaunchKernelGGL((act8_columns_kernel<KM>), dim3(p.S, p.tiles), dim3(256), 0, A8_ST, rows, M, K, p.across,             \
                     (const bf16*)dY, (int)dys, (const bf16*)X, (int)xs, out)
  if (K <= 4) A8_COLUMNS(4);
  else A8_COLUMNS(8);
#undef A8_COLUMNS
  PVN3D_LAUNCH_CHECK();
  return p.S > 1 ? rv::fold(p.S, count, count, (const float*)workspace, dW, nullptr, A8_ST) : 0;
}
