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
  float g[K][VEC], be[K][VEC], aw[K][VEC], ab[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = (k * TPR + t) * VEC + i;
      g[k][i] = c < C ? (w ? w[c] : 1.f) : 0.f;
      be[k][i] = c < C && b ? b[c] : 0.f;
      aw[k][i] = 0.f;
      ab[k][i] = 0.f;
    }
  const float rc = 1.f / (float)C;
  for (long long base = (long long)blockIdx.x * (RPB * R); base < rows; base += (long long)gridDim.x * (RPB * R)) {
    float v[R][K][VEC], d[R][K][VEC], mu[R], rs[R];
    unsigned bits[R][K];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long at = base + r * RPB + rg, row = at < rows ? at : rows - 1;
      mu[r] = mean[row];
      rs[r] = rstd[row];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + t) * VEC;
        rv::load_chunk<T>(dy + row * dys + c, C - c, d[r][k]);
        if (FROM8) {
          const bool in = c < C;
          rv::load_codes<VEC>(codes + row * pitch + (in ? c : 0), rv::group_step(scales[row * G + (in ? c / rv::GROUP : 0)]),
                              v[r][k]);
          bits[r][k] = mask ? (unsigned)mask[row * MB + (in ? c / 8 : 0)] >> (c & 7) : 0xffu;
        } else {
          rv::load_chunk<T>(x + row * xs + c, C - c, v[r][k]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * RPB + rg;
      const bool live = row < rows;
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const bool in = (k * TPR + t) * VEC + i < C;
          const float xh = in ? (v[r][k][i] - mu[r]) * rs[r] : 0.f;
          bool on = in && live;
          if (FROM8)
            on = on && ((bits[r][k] >> i) & 1u);
          else if (relu)
            on = on && fmaf(xh, g[k][i], be[k][i]) > 0.f;
          const float dz = on ? d[r][k][i] : 0.f;
          aw[k][i] = fmaf(dz, xh, aw[k][i]);
          ab[k][i] += dz;
          const float u = dz * g[k][i];
          s1 += u;
          s2 = fmaf(u, xh, s2);
          d[r][k][i] = u;
          v[r][k][i] = xh;
        }
      if (dx) {
        s1 = row_sum<TPR>(s1, red) * rc;
        s2 = row_sum<TPR>(s2, red) * rc;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = (k * TPR + t) * VEC;
          float o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            o[i] = c + i < C ? rs[r] * (d[r][k][i] - s1 - v[r][k][i] * s2) : 0.f;
          if (live && c < dxcols) rv::store_chunk<T>(dx + row * dxs + c, dxcols - c, o);
        }
      }
    }
  }
  if (!part) return;
  float* const pw = part + (size_t)blockIdx.x * 2 * C;
  if (TPR > 64) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (k * TPR + t) * VEC + i;
        if (c < C) {
          pw[c] = aw[k][i];
          pw[C + c] = ab[k][i];
        }
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
        for (int i = 0; i < VEC; ++i) fold[wave * COLS + (k * TPR + t) * VEC + i] = which ? ab[k][i] : aw[k][i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256)
      pw[which * C + c] = (fold[c] + fold[COLS + c]) + (fold[2 * COLS + c] + fold[3 * COLS + c]);
  }
}

// part [P][2 C] -> dw, db: 32 columns x 32 slices of P per workgroup, in a fixed order
__global__ __launch_bounds__(1024) void ln_grad_sum_kernel(int P, int C, const float* __restrict__ part,
                                                           float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float s[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
  float a = 0.f;
  if (col < 2 * C)
    for (int p = sl; p < P; p += 32) a += part[(size_t)p * 2 * C + col];
  s[sl][threadIdx.x & 31] = a;
  __syncthreads();
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    if (sl < o) s[sl][threadIdx.x & 31] += s[sl + o][threadIdx.x & 31];
    __syncthreads();
  }
  if (sl == 0 && col < 2 * C) (col < C ? dw[col] : db[col - C]) = s[0][threadIdx.x & 31];
}

// workgroups of a rows backward launch = its partial sums
int rows_grad_parts(int dtype, long long rows, int cover) {
  const long long n = ln::rows_blocks(rows, ln::rows_threads(cover, ln::vec_of(dtype)), 1);
  return (int)(n < ln::MAX_PARTS ? n : ln::MAX_PARTS);
}

template <typename T>
int rows_backward(int parts, long long rows, int C, const void* dy, long long dys, const void* x, long long xs,
                  const void* codes, long long pitch, const void* scales, const void* mask, const float* w, const float* b,
                  const float* mean, const float* rstd, int relu, void* dx, long long dxs, int dxcols, float* part,
                  hipStream_t st) {
  const int cover = C > dxcols ? C : dxcols;
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
  LN_ROWS_PICK(T, LN_CALL);
#undef LN_CALL
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

int ln::sum_parts(int parts, int C, const float* part, float* dw, float* db, hipStream_t st) {
  hipLaunchKernelGGL(ln_grad_sum_kernel, dim3(pvn3d_ceil_div(2 * C, 32)), dim3(1024), 0, st, parts, C, part, dw, db);
  PVN3D_LAUNCH_CHECK();
  return 0;
}

extern "C" size_t pvn3d_layer_norm_grad_workspace_bytes(int dtype, long long rows, int C, int cols) {
  if (rows <= 0 || C <= 0 || C > ln::MAX_C || dtype < 0 || dtype > 2) return 0;
  return (size_t)rows_grad_parts(dtype, rows, C > cols ? C : cols) * 2 * C * sizeof(float);
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
  if (!dx) dx_cols = C;
  const int parts = rows_grad_parts(dtype, rows, dx_cols);
  if (dweight && (!workspace || workspace_bytes < (size_t)parts * 2 * C * sizeof(float))) return (int)hipErrorInvalidValue;
  float* part = dweight ? (float*)workspace : nullptr;
  int rc;
  switch (dtype) {
    case 0: rc = rows_backward<float>(parts, rows, C, dy, dys, x, xs, codes, pitch, scales, mask, weight, bias, mean, rstd, relu, dx, dxs, dx_cols, part, (hipStream_t)stream); break;
    case 1: rc = rows_backward<bf16>(parts, rows, C, dy, dys, x, xs, codes, pitch, scales, mask, weight, bias, mean, rstd, relu, dx, dxs, dx_cols, part, (hipStream_t)stream); break;
    default: rc = rows_backward<fp16>(parts, rows, C, dy, dys, x, xs, codes, pitch, scales, mask, weight, bias, mean, rstd, relu, dx, dxs, dx_cols, part, (hipStream_t)stream); break;
  }
  if (rc || !dweight) return rc;
  return ln::sum_parts(parts, C, part, dweight, dbias, (hipStream_t)stream);
}
