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
// TPR threads share a row, chunk k of thread t = the VEC channels from (k TPR + t) VEC on (16 bytes): K chunks cover the
// row, R rows per thread are in flight at once.
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
  const int G = (C + rv::GROUP - 1) / rv::GROUP, MB = (C + 7) / 8;
  const ln::lane_cols<T, TPR, K> col(t, C);
  float g[K][VEC], be[K][VEC];
  col.params(w, 1.f, C, g);
  col.params(b, 0.f, C, be);
  const float rc = 1.f / (float)C, floor = relu ? 0.f : -__builtin_inff();
  for (long long base = (long long)blockIdx.x * (RPB * R); base < rows; base += (long long)gridDim.x * (RPB * R)) {
    float v[R][K][VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * RPB + rg;
      const T* const p = x + (row < rows ? row : rows - 1) * xs;
#pragma unroll
      for (int k = 0; k < K; ++k) col.load(p, k, C, v[r][k]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * RPB + rg;
      const bool live = row < rows;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s = fmaf(v[r][k][i], col.own[k][i], s);
      const float mu = row_sum<TPR>(s, red) * rc;
      float q = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = v[r][k][i] - mu;
          q = fmaf(d * col.own[k][i], d, q);
        }
      const float rs = 1.f / sqrtf(row_sum<TPR>(q, red) * rc + eps);
      if (live && t == 0) {
        mean[row] = mu;
        rstd[row] = rs;
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = col.c[k];
        float z[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i)       // (maximum: a NaN stays one, which max(z, 0) would make 0)
          z[i] = __builtin_elementwise_maximum(fmaf((v[r][k][i] - mu) * rs, g[k][i], be[k][i]), floor);
        if (live) col.store(y + row * ys, k, C, z);
        if (SAVE8) {
          constexpr int LPG = rv::GROUP / VEC < TPR ? rv::GROUP / VEC : TPR;       // lanes per group
          unsigned big = 0, wd[VEC / 4];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {                      // as integers: NaN is the largest
            const unsigned a = __float_as_uint(v[r][k][i]) & 0x7fffffffu;
            big = max(big, col.own[k][i] != 0.f ? a : 0u);
          }
          const unsigned sc = rv::group_scale(rv::lanes_max<LPG>(big));
          rv::group_codes<VEC>(v[r][k], sc, wd);
          if (live && c < C) {
            rv::store_codes(codes + row * pitch, c, col.skip[k], wd);
            if ((c & (rv::GROUP - 1)) == 0) scales[row * G + c / rv::GROUP] = (unsigned char)sc;
          }
          if (mask) {                                          // y is 0 or positive here: minus its bits, the sign bit
            unsigned bits = 0;
#pragma unroll
            for (int i = VEC - 1; i >= 0; --i) bits = __builtin_amdgcn_alignbit(bits, 0u - __float_as_uint(z[i]), 31);
            bits >>= col.skip[k];
            if (VEC == 4 && TPR > 1) {                         // two lanes share a byte
              const unsigned other = rv::dpp(bits, 1);
              bits |= c + 4 < C ? other << 4 : 0u;
            }
            if (live && c < C && (c & 7) == 0) mask[row * MB + c / 8] = (unsigned char)bits;
          }
        }
      }
      if (ycols > C && live)
        for (int c = C + t; c < ycols; c += TPR) traits<T>::store1(y + row * ys + c, 0.f);
    }
  }
}

template <typename T>
int rows_forward(long long rows, int C, const void* x, long long xs, const float* w, const float* b, float eps, int relu,
                 void* y, long long ys, int ycols, float* mean, float* rstd, void* codes, long long pitch, void* scales,
                 void* mask, hipStream_t st) {
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
  LN_ROWS_PICK(T, C, LN_CALL);
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
