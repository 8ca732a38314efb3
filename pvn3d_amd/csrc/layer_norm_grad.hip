// layer_norm_grad.hip -- the backward pass of layer_norm.hip over rows, and the sum of the partial weight gradients.
#include "layer_norm.h"

namespace {

using rv::bf16;
using rv::fp16;
using rv::traits;
using ln::row_sum;

// ------------------------------------------------------------------------------------------------ rows, backward
// As the forward; a thread's channels are the same for all its rows, so dw and db are summed in its registers over the
// rows of the workgroup, then over the workgroup's row slots (shuffles, LDS) into part[workgroup][2][C].
// Bound by HBM: dy and x read, dx written, once each.  bf16 786432 x 128: 115 us = 5.2 TB/s; 393216 x 196 from 8 bits: 100 us
// = 4.0 TB/s (25 of 32 lanes have a chunk; 8 small loads a row); the sum of the partials another 5 us.
// FROM8: code 2^e - mean is one fma (code 2^e is exact), with the rounding that x - mean has.
template <typename T, int TPR, int K, int R, bool FROM8>
__global__ __launch_bounds__(256) void ln_rows_grad_kernel(long long rows, int C, const T* __restrict__ dy, int dys,
                                                           const T* __restrict__ x, int xs,
                                                           const signed char* __restrict__ codes, int pitch,
                                                           const unsigned char* __restrict__ scales,
                                                           const unsigned char* __restrict__ mask,
                                                           const float* __restrict__ w, const float* __restrict__ b,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           int relu, T* __restrict__ dx, int dxs, int dxcols,
                                                           float* __restrict__ part_w, float* __restrict__ part_b,
                                                           size_t part_stride) {
  constexpr int VEC = traits<T>::VEC;
  constexpr int RPB = 256 / TPR;
  constexpr int COLS = TPR * K * VEC;
  __shared__ float red[4];
  __shared__ float fold[TPR > 64 ? 1 : 4 * COLS];
  const int t = threadIdx.x % TPR, rg = threadIdx.x / TPR;
  const int G = (C + rv::GROUP - 1) / rv::GROUP, MB = (C + 7) / 8;
  const bool ragged = (C & (VEC - 1)) != 0;
  const ln::lane_cols<T, TPR, K> col(t, C);
  float g[K][VEC], be[K][VEC], aw[K][VEC], ab[K][VEC];
  col.params(w, 1.f, C, g);
  col.params(b, 0.f, C, be);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      aw[k][i] = 0.f;
      ab[k][i] = 0.f;
    }
  const float rc = 1.f / (float)C;
  for (long long base = (long long)blockIdx.x * (RPB * R); base < rows; base += (long long)gridDim.x * (RPB * R)) {
    const int last = (int)(rows - 1 - base < RPB * R - 1 ? rows - 1 - base : RPB * R - 1);
    const T* const db = dy + base * dys;
    const T* const xb = x + base * xs;
    T* const ob = dx + base * dxs;
    const signed char* const cb = codes + base * pitch;
    const unsigned char* const sb = scales + base * G;
    const unsigned char* const mb = mask + base * MB;
    rv::u4_any rx[R][K], rd[R][K];
    float mu[R], rs[R];
    unsigned cw[R][K][VEC / 4];
    unsigned char sc[R][K][2], mk[R][K][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int rl = min(rg + r * RPB, last);
      mu[r] = *rv::at32(mean + base, rl * 4u);
      rs[r] = *rv::at32(rstd + base, rl * 4u);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        rd[r][k] = col.load(db, __umul24(rl, dys), k, C);
        if (FROM8) {
          // a window that repeats values of its neighbour may start in the group before its own
          const int c = min(col.c[k], (C - 1) & ~(VEC - 1)), at = col.at[k];
          const unsigned srow = __umul24(rl, G), mrow = __umul24(rl, MB);
          rv::load_codes(rv::at32(cb, __umul24(rl, pitch) + at), cw[r][k]);
          sc[r][k][0] = *rv::at32(sb, srow + c / rv::GROUP);
          if (ragged) sc[r][k][1] = *rv::at32(sb, srow + at / rv::GROUP);
          if (mask) mk[r][k][0] = *rv::at32(mb, mrow + at / 8);
          if (mask && ragged) mk[r][k][1] = *rv::at32(mb, mrow + min(at / 8 + 1, MB - 1));
        } else {
          rx[r][k] = col.load(xb, __umul24(rl, xs), k, C);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);       // all loads on their way before anything waits for one
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int rl = rg + r * RPB;
      const bool live = rl <= last;
      float v[K][VEC], d[K][VEC], s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        traits<T>::unpack(rd[r][k], d[k]);
        if (!FROM8) traits<T>::unpack(rx[r][k], v[k]);
        const float a = FROM8 ? rv::group_step(sc[r][k][0]) : 0.f, a0 = FROM8 && ragged ? rv::group_step(sc[r][k][1]) : a;
        unsigned bits = 0xffffffffu;
        if (FROM8 && mask) bits = ((unsigned)mk[r][k][0] | (ragged ? (unsigned)mk[r][k][1] << 8 : 0u)) >> (col.at[k] & 7);
        if (FROM8 && !live) bits = 0u;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xm = FROM8 ? fmaf(rv::code_at(cw[r][k], i), i < col.skip[k] ? a0 : a, -mu[r]) : v[k][i] - mu[r];
          const float xh = xm * rs[r];
          float dz;
          if (FROM8) {
            // bit i as a mask of the whole word
            const unsigned on = (unsigned)__builtin_amdgcn_sbfe((int)bits, i, 1);
            dz = __uint_as_float(__float_as_uint(d[k][i]) & on);
          } else {
            const bool off_ = relu && fmaf(xh, g[k][i], be[k][i]) <= 0.f;          // (a NaN passes, as in the forward)
            dz = live && !off_ ? d[k][i] : 0.f;
          }
          aw[k][i] = fmaf(dz, xh, aw[k][i]);
          ab[k][i] += dz;
          const float u = dz * g[k][i], um = u * col.own[k][i];
          s1 += um;
          s2 = fmaf(um, xh, s2);
          d[k][i] = u;
          v[k][i] = xh;
        }
      }
      if (dx) {
        s1 = row_sum<TPR>(s1, red) * rc;
        s2 = row_sum<TPR>(s2, red) * rc;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] = rs[r] * (d[k][i] - s1 - v[k][i] * s2);
          if (live) col.store(ob, __umul24(rl, dxs), k, C, o);
        }
        if (dxcols > C && live)
#pragma unroll 1
          for (int c = C + t; c < dxcols; c += TPR)
            traits<T>::store1(rv::at32(ob, (__umul24(rl, dxs) + c) * (unsigned)sizeof(T)), 0.f);
      }
    }
  }
  if (!part_w) return;
  float* const pw = part_w + blockIdx.x * part_stride;
  float* const pb = part_b + blockIdx.x * part_stride;
  if (TPR > 64) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (col.own[k][i] != 0.f) {
          pw[col.at[k] + i] = aw[k][i];
          pb[col.at[k] + i] = ab[k][i];
        }
    return;
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i)
#pragma unroll
      for (int o = TPR; o < 64; o <<= 1) {
        aw[k][i] += __shfl_xor(aw[k][i], o, 64);
        ab[k][i] += __shfl_xor(ab[k][i], o, 64);
      }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    if (lane < TPR) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (col.own[k][i] != 0.f) fold[wave * COLS + col.at[k] + i] = which ? ab[k][i] : aw[k][i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256)
      (which ? pb : pw)[c] = (fold[c] + fold[COLS + c]) + (fold[2 * COLS + c] + fold[3 * COLS + c]);
  }
}

// Workgroups of a rows backward launch = its partial sums: what the registers let stay on the chip (`resident` a CU), each
// with four rows at least where it takes a row at a time.  bf16 16384 x 4096: 100 us,
// 125 with twice as many, 137 with 2048; 46000 x 753: 45, 51, 57; 2000 x 1536: 19, 19, 36; 786432 x 128: 119, 122, 122.
// A call of a few passes' rows is one workgroup's, which writes dw and db itself (no second launch).
int rows_grad_parts(int dtype, long long rows, int C, bool from8) {
  const int vec = ln::vec_of(dtype), tpr = ln::rows_threads(C, vec), k = (C + tpr * vec - 1) / (tpr * vec);
  int resident;
  if (vec == 8) resident = k == 1 ? 4 : k == 2 ? 3 : 1;
  else resident = k == 1 ? 8 - from8 : k == 2 ? (tpr == 64 ? 5 : 5 - from8) : k <= 4 ? 2 : 1;
  if (ln::rows_blocks(rows, tpr, 1) <= 8) return 1;
  const long long n = tpr == 256 ? (rows + 3) / 4 : ln::rows_blocks(rows, tpr, k == 1 ? 2 : 1);
  return (int)(n < 256 * resident ? n : 256 * resident);
}

template <typename T>
int rows_backward(int parts, long long rows, int C, const void* dy, long long dys, const void* x, long long xs,
                  const void* codes, long long pitch, const void* scales, const void* mask, const float* w, const float* b,
                  const float* mean, const float* rstd, int relu, void* dx, long long dxs, int dxcols, float* pw, float* pb,
                  size_t ps, hipStream_t st) {
#define LN_CALL(T, TPR, K, R)                                                                                            \
  do {                                                                                                                   \
    if (codes)                                                                                                           \
      hipLaunchKernelGGL((ln_rows_grad_kernel<T, TPR, K, R, true>), dim3(parts), dim3(256), 0, st, rows, C,              \
                         (const T*)dy, (int)dys, (const T*)nullptr, 0, (const signed char*)codes, (int)pitch,            \
                         (const unsigned char*)scales, (const unsigned char*)mask, w, b, mean, rstd, relu, (T*)dx,       \
                         (int)dxs, dxcols, pw, pb, ps);                                                                  \
    else                                                                                                                 \
      hipLaunchKernelGGL((ln_rows_grad_kernel<T, TPR, K, R, false>), dim3(parts), dim3(256), 0, st, rows, C,             \
                         (const T*)dy, (int)dys, (const T*)x, (int)xs, (const signed char*)nullptr, 0,                   \
                         (const unsigned char*)nullptr, (const unsigned char*)nullptr, w, b, mean, rstd, relu, (T*)dx,   \
                         (int)dxs, dxcols, pw, pb, ps);                                                                  \
  } while (0)
  LN_ROWS_PICK(T, C, LN_CALL);
#undef LN_CALL
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" size_t pvn3d_layer_norm_grad_workspace_bytes(int dtype, long long rows, int C) {
  if (rows <= 0 || C <= 0 || C > ln::MAX_C || dtype < 0 || dtype > 2) return 0;
  const int parts = rows_grad_parts(dtype, rows, C, false);            // (from 8 bits: as many or fewer)
  return parts > 1 ? (size_t)parts * 2 * C * sizeof(float) : 0;
}
extern "C" int pvn3d_layer_norm_grad(int dtype, long long rows, int C, const void* dy, long long dys, const void* x,
                                     long long xs, const void* codes, long long pitch, const void* scales,
                                     const void* mask, const float* weight, const float* bias, const float* mean,
                                     const float* rstd, int relu, void* dx, long long dxs, int dx_cols, float* dweight,
                                     float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype < 0 || dtype > 2 || C <= 0 || C > ln::MAX_C || dys < 0 || xs < 0) return (int)hipErrorInvalidValue;
  if (dys > ln::MAX_STRIDE || xs > ln::MAX_STRIDE || dxs > ln::MAX_STRIDE || pitch > ln::MAX_STRIDE)
    return (int)hipErrorInvalidValue;
  if (dx && (dx_cols < C || dx_cols > C + 15 || dxs < dx_cols)) return (int)hipErrorInvalidValue;
  if ((dweight == nullptr) != (dbias == nullptr) || (!dx && !dweight)) return (int)hipErrorInvalidValue;
  if (codes && (!scales || (pitch & 15) || pitch < C || (relu != 0) != (mask != nullptr))) return (int)hipErrorInvalidValue;
  if (rows <= 0) {
    if (dweight) {
      pvn3d_fill_u32(dweight, 0, C, (hipStream_t)stream);
      pvn3d_fill_u32(dbias, 0, C, (hipStream_t)stream);
      PVN3D_LAUNCH_CHECK();
    }
    return 0;
  }
  if (!dy || (!x && !codes) || !mean || !rstd) return (int)hipErrorInvalidValue;
  const int parts = rows_grad_parts(dtype, rows, C, codes != nullptr);
  if (dweight && parts > 1 && (!workspace || workspace_bytes < (size_t)parts * 2 * C * sizeof(float)))
    return (int)hipErrorInvalidValue;
  float* const part = (float*)workspace;
  float* const pw = !dweight ? nullptr : parts > 1 ? part : dweight;
  float* const pb = !dweight ? nullptr : parts > 1 ? part + C : dbias;
  const size_t ps = parts > 1 ? 2 * (size_t)C : 0;
  const auto run = dtype == 0 ? rows_backward<float> : dtype == 1 ? rows_backward<bf16> : rows_backward<fp16>;
  const int rc = run(parts, rows, C, dy, dys, x, xs, codes, pitch, scales, mask, weight, bias, mean, rstd, relu, dx, dxs,
                     dx_cols, pw, pb, ps, (hipStream_t)stream);
  if (rc || !dweight || parts == 1) return rc;
  return rv::fold(parts, 2 * (size_t)C, C, part, dweight, dbias, (hipStream_t)stream);
}
