// layer_norm.hip -- layer norm over the channels of every point, forward and backward (gfx950).
//
// Stands beside the BatchNorm passes of mlp_train.hip: [1x1 convolution -> norm -> ReLU] with statistics of the point's own
// channels instead of the batch's (a rank that trains on one frame has the same arithmetic as one that trains on 24).
//   mean = sum_c x / C,  var = sum_c (x - mean)^2 / C,  rstd = 1 / sqrt(var + eps),  xh = (x - mean) rstd
//   z = w xh + b,  y = z or max(z, 0)
// backward, with dz = dy [z > 0] (or dy), u = w dz:
//   dx = rstd (u - sum(u) / C - xh sum(u xh) / C),  dw = sum_points dz xh,  db = sum_points dz
// Statistics, sums and all arithmetic in fp32 whatever the type of x; one rounding, at the store.  The variance is taken
// about the mean from the values held in registers (two passes over registers, one over memory).
//
// Two layouts.  ROWS: [rows][C], C contiguous.  CHANNELS: (B, C, M), M contiguous -- the module API's feature tensors.
// The rows kernels can put x away in the 8-bit group form of rowvec.h in the same pass (and, with a ReLU, one bit
// per value for z > 0), and the backward pass can take it from there: it then reads 1 byte per value instead of 2 or 4.
#include "layer_norm.h"

namespace {

using rv::bf16;
using rv::fp16;
using rv::traits;
using ln::row_sum;

// ------------------------------------------------------------------------------------------------ rows, forward
// TPR threads share a row, chunk k of thread t = channels (k TPR + t) VEC ..: K chunks cover the row, R rows per thread
// are in flight at once.
template <typename T, int TPR, int K, int R, bool SAVE8>
__global__ __launch_bounds__(256) void ln_rows_kernel(long long rows, int C, const T* __restrict__ x, long long xs,
                                                      const float* __restrict__ w, const float* __restrict__ b, float eps,
                                                      int relu, T* __restrict__ y, long long ys, int ycols,
                                                      float* __restrict__ mean, float* __restrict__ rstd,
                                                      signed char* __restrict__ codes, long long pitch,
                                                      unsigned char* __restrict__ scales,
                                                      unsigned char* __restrict__ mask) {
  constexpr int VEC = traits<T>::VEC;
  constexpr int RPB = 256 / TPR;
  __shared__ float red[4];
  const int t = threadIdx.x % TPR, rg = threadIdx.x / TPR;
  float g[K][VEC], be[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = (k * TPR + t) * VEC + i;
      g[k][i] = c < C ? (w ? w[c] : 1.f) : 0.f;
      be[k][i] = c < C && b ? b[c] : 0.f;
    }
  const float rc = 1.f / (float)C;
  for (long long base = (long long)blockIdx.x * (RPB * R); base < rows; base += (long long)gridDim.x * (RPB * R)) {
    float v[R][K][VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * RPB + rg;
      const T* p = x + (row < rows ? row : rows - 1) * xs;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + t) * VEC;
        rv::load_chunk<T>(p + c, C - c, v[r][k]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * RPB + rg;
      const bool live = row < rows;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s += v[r][k][i];
      const float mu = row_sum<TPR>(s, red) * rc;
      float q = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = (k * TPR + t) * VEC + i < C ? v[r][k][i] - mu : 0.f;
          q = fmaf(d, d, q);
        }
      const float rs = 1.f / sqrtf(row_sum<TPR>(q, red) * rc + eps);
      if (live && t == 0) {
        mean[row] = mu;
        rstd[row] = rs;
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + t) * VEC;
        float z[VEC];
        unsigned bits = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          z[i] = fmaf((v[r][k][i] - mu) * rs, g[k][i], be[k][i]);
          bits |= (z[i] > 0.f ? 1u : 0u) << i;
          // (a NaN stays one: max(z, 0) would make it 0)
          if (relu) z[i] = z[i] < 0.f ? 0.f : z[i];
          if (c + i >= C) z[i] = 0.f;
        }
        if (live && c < ycols) rv::store_chunk<T>(y + row * ys + c, ycols - c, z);
        if (SAVE8) {
          constexpr int LPG = rv::GROUP / VEC < TPR ? rv::GROUP / VEC : TPR;       // lanes per group
          const unsigned sc = rv::lanes_scale<VEC, LPG>(v[r][k]);
          if (live && c < C) {
            rv::store_codes<VEC>(codes + row * pitch + c, v[r][k], rv::group_inverse(sc));
            if ((c & (rv::GROUP - 1)) == 0) scales[row * ((C + rv::GROUP - 1) / rv::GROUP) + c / rv::GROUP] = (unsigned char)sc;
          }
          if (mask) {
            unsigned other = 0;
            if (VEC == 4) other = (unsigned)__shfl_down((int)bits, 1, 64);          // two lanes share a byte
            if (live && c < C && (c & 7) == 0)
              mask[row * ((C + 7) / 8) + c / 8] = (unsigned char)(bits | (VEC == 4 ? (c + 4 < C && TPR > 1 ? other << 4 : 0u) : 0u));
          }
        }
      }
    }
  }
}

template <typename T>
int rows_forward(long long rows, int C, const void* x, long long xs, const float* w, const float* b, float eps, int relu,
                 void* y, long long ys, int ycols, float* mean, float* rstd, void* codes, long long pitch, void* scales,
                 void* mask, hipStream_t st) {
  const int cover = C > ycols ? C : ycols;
#define LN_CALL(T, TPR, K, R)                                                                                           \
  do {                                                                                                                  \
    const long long nb = ln::rows_blocks(rows, TPR, R);                                                                     \
    const dim3 grid((unsigned)(nb < 16384 ? nb : 16384));                                                               \
    if (codes)                                                                                                          \
      hipLaunchKernelGGL((ln_rows_kernel<T, TPR, K, R, true>), grid, dim3(256), 0, st, rows, C, (const T*)x, xs, w, b, \
                         eps, relu, (T*)y, ys, ycols, mean, rstd, (signed char*)codes, pitch, (unsigned char*)scales,   \
                         (unsigned char*)mask);                                                                         \
    else                                                                                                                \
      hipLaunchKernelGGL((ln_rows_kernel<T, TPR, K, R, false>), grid, dim3(256), 0, st, rows, C, (const T*)x, xs, w, b, \
                         eps, relu, (T*)y, ys, ycols, mean, rstd, nullptr, 0ll, nullptr, nullptr);                      \
  } while (0)
  LN_ROWS_PICK(T, LN_CALL);
#undef LN_CALL
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int pvn3d_layer_norm(int dtype, long long rows, int C, const void* x, long long xs, const float* weight,
                                const float* bias, float eps, int relu, void* y, long long ys, int y_cols, float* mean,
                                float* rstd, void* codes, long long pitch, void* scales, void* mask, void* stream) {
  if (dtype < 0 || dtype > 2 || C <= 0 || C > ln::MAX_C || y_cols < C || y_cols > C + 15 || ys < y_cols || xs < 0)
    return (int)hipErrorInvalidValue;
  if (codes && (!scales || (pitch & 15) || pitch < C)) return (int)hipErrorInvalidValue;
  if (rows <= 0) return 0;
  if (!x || !y || !mean || !rstd) return (int)hipErrorInvalidValue;
  switch (dtype) {
    case 0: return rows_forward<float>(rows, C, x, xs, weight, bias, eps, relu, y, ys, y_cols, mean, rstd, codes, pitch, scales, mask, (hipStream_t)stream);
    case 1: return rows_forward<bf16>(rows, C, x, xs, weight, bias, eps, relu, y, ys, y_cols, mean, rstd, codes, pitch, scales, mask, (hipStream_t)stream);
    default: return rows_forward<fp16>(rows, C, x, xs, weight, bias, eps, relu, y, ys, y_cols, mean, rstd, codes, pitch, scales, mask, (hipStream_t)stream);
  }
}
