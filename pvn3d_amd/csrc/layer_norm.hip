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

// Bound by HBM: x read once, y written once.  bf16 1572864 x 64: 68 us = 5.9 TB/s (a large copy on this card: 4.9);
// 393216 x 196 with x put away in 8 bits and ReLU bits, 78 us = 5.1 TB/s (lanes behind the row's end and the codes'
// arithmetic cost the rest).  128 x 512, a call whose cost is its launch: 3.6 us.  What it took: the parameters loaded in
// vectors (with a load per value 98304 x 1024 took 237 us, now 74), the loads of both rows ahead of any wait, addresses as a
// shared base plus 32-bit offsets instead of a 64-bit product per row and tensor, sums over lanes in registers.
// ------------------------------------------------------------------------------------------------ rows, forward
// TPR threads share a row, chunk k of thread t = the VEC channels from (k TPR + t) VEC on (16 bytes): K chunks cover the
// row, R rows per thread are in flight at once.
template <typename T, int TPR, int K, int R, bool SAVE8, bool STREAM>
__global__ __launch_bounds__(256) void ln_rows_kernel(long long rows, int C, const T* __restrict__ x, int xs,
                                                      const float* __restrict__ w, const float* __restrict__ b, float eps,
                                                      int relu, T* __restrict__ y, int ys, int ycols,
                                                      float* __restrict__ mean, float* __restrict__ rstd,
                                                      signed char* __restrict__ codes, int pitch,
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
  const float rc = 1.f / (float)C;
  float low = relu ? 0.f : -__builtin_inff();
  asm("" : "+v"(low));             // a register, not a choice of two constants at every use
  for (long long base = (long long)blockIdx.x * (RPB * R); base < rows; base += (long long)gridDim.x * (RPB * R)) {
    const int last = (int)(rows - 1 - base < RPB * R - 1 ? rows - 1 - base : RPB * R - 1);
    const T* const xb = x + base * xs;
    T* const yb = y + base * ys;
    signed char* const cb = codes + base * pitch;
    unsigned char* const sb = scales + base * G;
    unsigned char* const mb = mask + base * MB;
    rv::u4_any raw[R][K];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned row = __umul24(min(rg + r * RPB, last), xs);
#pragma unroll
      for (int k = 0; k < K; ++k) raw[r][k] = col.template load<STREAM>(xb, row, k, C);
    }
    __builtin_amdgcn_sched_barrier(0);       // all loads on their way before anything waits for one
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int rl = rg + r * RPB;
      const bool live = rl <= last;
      float v[K][VEC], s = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        traits<T>::unpack(raw[r][k], v[k]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s = fmaf(v[k][i], col.own[k][i], s);
      }
      const float mu = row_sum<TPR>(s, red) * rc;
      float q = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = v[k][i] - mu;
          q = fmaf(d * col.own[k][i], d, q);
        }
      const float rs = __builtin_amdgcn_rsqf(fmaf(row_sum<TPR>(q, red), rc, eps));      // v_rsq_f32: within one ulp
      if (live && t == 0) {
        *rv::at32(mean + base, rl * 4u) = mu;
        *rv::at32(rstd + base, rl * 4u) = rs;
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = col.c[k];
        float z[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i)       // (maximum: a NaN stays one, which max(z, 0) would make 0)
          z[i] = __builtin_elementwise_maximum(fmaf((v[k][i] - mu) * rs, g[k][i], be[k][i]), low);
        if (live) col.template store<STREAM>(yb, __umul24(rl, ys), k, C, z);
        if (SAVE8) {
          constexpr int LPG = rv::GROUP / VEC < TPR ? rv::GROUP / VEC : TPR;       // lanes per group
          unsigned big = 0, wd[VEC / 4];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {                      // as integers: NaN is the largest
            const unsigned a = __float_as_uint(v[k][i]) & 0x7fffffffu;
            big = max(big, col.own[k][i] != 0.f ? a : 0u);
          }
          const unsigned sc = rv::group_scale(rv::lanes_max<LPG>(big));
          rv::group_codes<VEC>(v[k], sc, wd);
          if (live && c < C) {
            rv::store_codes(rv::at32(cb, __umul24(rl, pitch) + c), col.skip[k], wd);
            if ((c & (rv::GROUP - 1)) == 0) *rv::at32(sb, __umul24(rl, G) + c / rv::GROUP) = (unsigned char)sc;
          }
          if (mask) {           // y is +0, positive or a NaN of either sign: any bit of it carries into the sign, and stays there
            unsigned bits = 0;
#pragma unroll
            for (int i = VEC - 1; i >= 0; --i)
              bits = __builtin_amdgcn_alignbit(bits, __builtin_elementwise_add_sat(__float_as_uint(z[i]), 0x7fffffffu), 31);
            bits >>= col.skip[k];
            if (VEC == 4 && TPR > 1) {                         // two lanes share a byte
              const unsigned other = rv::dpp(bits, 1);
              bits |= c + 4 < C ? other << 4 : 0u;
            }
            if (live && c < C && (c & 7) == 0) *rv::at32(mb, __umul24(rl, MB) + c / 8) = (unsigned char)bits;
          }
        }
      }
      if (ycols > C && live)
#pragma unroll 1
        for (int c = C + t; c < ycols; c += TPR)
          traits<T>::store1(rv::at32(yb, (__umul24(rl, ys) + c) * (unsigned)sizeof(T)), 0.f);
    }
  }
}

// Workgroups of a forward launch: enough to keep every CU busy, few enough that loading the parameters is spread over several
// rows, and all with as many passes.  bf16 786432 x 128 with the input saved: 96 us with two passes each, 99 with three; where
// a workgroup takes four rows or two at a time 46000 x 753 29 us with two or three passes each, 34 with one, 31 with two in
// some and one in others; 150000 x 600 70 us with five, 73 with ten.
constexpr long long most_blocks(int tpr, int k) { return tpr <= 64 && k == 1 ? 12288 : 8192; }

// R8: two rows in flight where the input is saved and a row is two chunks a lane (bf16 46000 x 753: 49 us, 52 with one;
// without saving 150000 x 600 73 us, 70 with one)
template <typename T>
int rows_forward(long long rows, int C, const void* x, long long xs, const float* w, const float* b, float eps, int relu,
                 void* y, long long ys, int ycols, float* mean, float* rstd, void* codes, long long pitch, void* scales,
                 void* mask, hipStream_t st) {
  const bool stream = rows * C * (long long)sizeof(T) >= rv::STREAM_BYTES;
#define LN_ONE(T, TPR, K, R, SAVE8, STREAM)                                                                              \
  hipLaunchKernelGGL((ln_rows_kernel<T, TPR, K, R, SAVE8, STREAM>), grid, dim3(256), 0, st, rows, C, (const T*)x, (int)xs, \
                     w, b, eps, relu, (T*)y, (int)ys, ycols, mean, rstd, (signed char*)codes, (int)pitch,               \
                     (unsigned char*)scales, (unsigned char*)mask)
#define LN_CALL(T, TPR, K, R)                                                                                           \
  do {                                                                                                                  \
    constexpr int R8 = K == 2 ? 2 : R;                                                                                  \
    const long long nb = ln::rows_blocks(rows, TPR, codes ? R8 : R);                                                    \
    const dim3 grid(rv::even_grid(nb, most_blocks(TPR, K)));                                                            \
    if (codes && stream) LN_ONE(T, TPR, K, R8, true, true);                                                             \
    else if (codes) LN_ONE(T, TPR, K, R8, true, false);                                                                 \
    else if (stream) LN_ONE(T, TPR, K, R, false, true);                                                                 \
    else LN_ONE(T, TPR, K, R, false, false);                                                                            \
  } while (0)
  LN_ROWS_PICK(T, C, LN_CALL);
#undef LN_CALL
#undef LN_ONE
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int pvn3d_layer_norm(int dtype, long long rows, int C, const void* x, long long xs, const float* weight,
                                const float* bias, float eps, int relu, void* y, long long ys, int y_cols, float* mean,
                                float* rstd, void* codes, long long pitch, void* scales, void* mask, void* stream) {
  if (dtype < 0 || dtype > 2 || C <= 0 || C > ln::MAX_C || y_cols < C || y_cols > C + 15 || ys < y_cols || xs < 0)
    return (int)hipErrorInvalidValue;
  if (xs > ln::MAX_STRIDE || ys > ln::MAX_STRIDE || pitch > ln::MAX_STRIDE) return (int)hipErrorInvalidValue;
  if (codes && (!scales || (pitch & 15) || pitch < C || (mask && !relu))) return (int)hipErrorInvalidValue;
  if (rows <= 0) return 0;
  if (!x || !y || !mean || !rstd) return (int)hipErrorInvalidValue;
  const auto run = dtype == 0 ? rows_forward<float> : dtype == 1 ? rows_forward<bf16> : rows_forward<fp16>;
  return run(rows, C, x, xs, weight, bias, eps, relu, y, ys, y_cols, mean, rstd, codes, pitch, scales, mask,
             (hipStream_t)stream);
}
