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
// FROM8: code 2^e - mean is one fma (code 2^e is exact), with the rounding that x - mean has.
template <typename T, int TPR, int K, int R, bool FROM8>
__global__ __launch_bounds__(256) void ln_rows_grad_kernel(long long rows, int C, const T* __restrict__ dy, long long dys,
                                                           const T* __restrict__ x, long long xs,
                                                           const signed char* __restrict__ codes, long long pitch,
                                                           const unsigned char* __restrict__ scales,
                                                           const unsigned char* __restrict__ mask,
                                                           const float* __restrict__ w, const float* __restrict__ b,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           int relu, T* __restrict__ dx, long long dxs, int dxcols,
                                                           float* __restrict__ part) {
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
    float v[R][K][VEC], d[R][K][VEC], mu[R], rs[R];
    unsigned cw[R][K][VEC / 4], bits[R][K];
    float step[R][K], step0[R][K];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long at = base + r * RPB + rg, row = at < rows ? at : rows - 1;
      mu[r] = mean[row];
      rs[r] = rstd[row];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        col.load(dy + row * dys, k, C, d[r][k]);
        if (FROM8) {
          // a window that repeats values of its neighbour may start in the group before its own
          const int c = min(col.c[k], (C - 1) & ~(VEC - 1)), at = col.at[k];
          rv::load_codes(codes + row * pitch + at, cw[r][k]);
          step[r][k] = rv::group_step(scales[row * G + c / rv::GROUP]);
          step0[r][k] = ragged ? rv::group_step(scales[row * G + at / rv::GROUP]) : step[r][k];
          bits[r][k] = 0xffffffffu;
          if (mask) {
            bits[r][k] = mask[row * MB + at / 8];
            if (ragged) bits[r][k] |= (unsigned)mask[row * MB + min(at / 8 + 1, MB - 1)] << 8;
            bits[r][k] >>= at & 7;
          }
        } else {
          col.load(x + row * xs, k, C, v[r][k]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * RPB + rg;
      const bool live = row < rows;
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float a = FROM8 ? step[r][k] : 0.f, a0 = FROM8 ? step0[r][k] : 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xm = FROM8 ? fmaf(rv::code_at(cw[r][k], i), i < col.skip[k] ? a0 : a, -mu[r]) : v[r][k][i] - mu[r];
          const float xh = xm * rs[r];
          float dz;
          if (FROM8) {
            // bit i as a mask of the whole word
            const unsigned on = (unsigned)__builtin_amdgcn_sbfe((int)(live ? bits[r][k] : 0u), i, 1);
            dz = __uint_as_float(__float_as_uint(d[r][k][i]) & on);
          } else {
            const bool off_ = relu && fmaf(xh, g[k][i], be[k][i]) <= 0.f;          // (a NaN passes, as in the forward)
            dz = live && !off_ ? d[r][k][i] : 0.f;
          }
          aw[k][i] = fmaf(dz, xh, aw[k][i]);
          ab[k][i] += dz;
          const float u = dz * g[k][i], um = u * col.own[k][i];
          s1 += um;
          s2 = fmaf(um, xh, s2);
          d[r][k][i] = u;
          v[r][k][i] = xh;
        }
      }
      if (dx) {
        s1 = row_sum<TPR>(s1, red) * rc;
        s2 = row_sum<TPR>(s2, red) * rc;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] = rs[r] * (d[r][k][i] - s1 - v[r][k][i] * s2);
          if (live) col.store(dx + row * dxs, k, C, o);
        }
        if (dxcols > C && live)
          for (int c = C + t; c < dxcols; c += TPR) traits<T>::store1(dx + row * dxs + c, 0.f);
      }
    }
  }
  if (!part) return;
  float* const pw = part + (size_t)blockIdx.x * 2 * C;
  if (TPR > 64) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (col.own[k][i] != 0.f) {
          pw[col.at[k] + i] = aw[k][i];
          pw[C + col.at[k] + i] = ab[k][i];
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
      pw[which * C + c] = (fold[c] + fold[COLS + c]) + (fold[2 * COLS + c] + fold[3 * COLS + c]);
  }
}

// workgroups of a rows backward launch = its partial sums
int rows_grad_parts(int dtype, long long rows, int C) {
  const long long n = ln::rows_blocks(rows, ln::rows_threads(C, ln::vec_of(dtype)), 1);
  return (int)(n < ln::MAX_PARTS ? n : ln::MAX_PARTS);
}

template <typename T>
int rows_backward(int parts, long long rows, int C, const void* dy, long long dys, const void* x, long long xs,
                  const void* codes, long long pitch, const void* scales, const void* mask, const float* w, const float* b,
                  const float* mean, const float* rstd, int relu, void* dx, long long dxs, int dxcols, float* part,
                  hipStream_t st) {
#define LN_CALL(T, TPR, K, R)                                                                                            \
  do {                                                                                                                   \
    if (codes)                                                                                                           \
      hipLaunchKernelGGL((ln_rows_grad_kernel<T, TPR, K, R, true>), dim3(parts), dim3(256), 0, st, rows, C,              \
                         (const T*)dy, dys, (const T*)nullptr, 0ll, (const signed char*)codes, pitch,                    \
                         (const unsigned char*)scales, (const unsigned char*)mask, w, b, mean, rstd, relu, (T*)dx, dxs,  \
                         dxcols, part);                                                                                  \
    else                                                                                                                 \
      hipLaunchKernelGGL((ln_rows_grad_kernel<T, TPR, K, R, false>), dim3(parts), dim3(256), 0, st, rows, C,             \
                         (const T*)dy, dys, (const T*)x, xs, (const signed char*)nullptr, 0ll,                           \
                         (const unsigned char*)nullptr, (const unsigned char*)nullptr, w, b, mean, rstd, relu, (T*)dx,   \
                         dxs, dxcols, part);                                                                             \
  } while (0)
  LN_ROWS_PICK(T, C, LN_CALL);
#undef LN_CALL
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" size_t pvn3d_layer_norm_grad_workspace_bytes(int dtype, long long rows, int C) {
  if (rows <= 0 || C <= 0 || C > ln::MAX_C || dtype < 0 || dtype > 2) return 0;
  return (size_t)rows_grad_parts(dtype, rows, C) * 2 * C * sizeof(float);
}
extern "C" int pvn3d_layer_norm_grad(int dtype, long long rows, int C, const void* dy, long long dys, const void* x,
                                     long long xs, const void* codes, long long pitch, const void* scales,
                                     const void* mask, const float* weight, const float* bias, const float* mean,
                                     const float* rstd, int relu, void* dx, long long dxs, int dx_cols, float* dweight,
                                     float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype < 0 || dtype > 2 || C <= 0 || C > ln::MAX_C || dys < 0 || xs < 0) return (int)hipErrorInvalidValue;
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
  const int parts = rows_grad_parts(dtype, rows, C);
  if (dweight && (!workspace || workspace_bytes < (size_t)parts * 2 * C * sizeof(float))) return (int)hipErrorInvalidValue;
  float* part = dweight ? (float*)workspace : nullptr;
  int rc;
  switch (dtype) {
    case 0: rc = rows_backward<float>(parts, rows, C, dy, dys, x, xs, codes, pitch, scales, mask, weight, bias, mean, rstd, relu, dx, dxs, dx_cols, part, (hipStream_t)stream); break;
    case 1: rc = rows_backward<bf16>(parts, rows, C, dy, dys, x, xs, codes, pitch, scales, mask, weight, bias, mean, rstd, relu, dx, dxs, dx_cols, part, (hipStream_t)stream); break;
    default: rc = rows_backward<fp16>(parts, rows, C, dy, dys, x, xs, codes, pitch, scales, mask, weight, bias, mean, rstd, relu, dx, dxs, dx_cols, part, (hipStream_t)stream); break;
  }
  if (rc || !dweight) return rc;
  return rv::fold(parts, 2 * (size_t)C, C, part, dweight, dbias, (hipStream_t)stream);
}
