// layer_norm_grad.hip -- the backward pass of layer_norm.hip over rows, and the sum of the partial weight gradients.
#include "layer_norm.h"

namespace {

using rv::bf16;
using rv::fp16;
using rv::traits;
using ln::row_sum;

constexpr int ACROSS = 2;                            // chunks across of a column workgroup

// ------------------------------------------------------------------------------------------------ rows, backward
// As the forward; a thread's channels are the same for all its rows, so dw and db are summed in its registers over the
// rows of the workgroup, then over the workgroup's row slots (shuffles, LDS) into part[workgroup][2][C].
// Bound by HBM: dy and x read, dx written, once each.  bf16 786432 x 128: 104 us = 5.8 TB/s; 393216 x 196 from 8 bits: 88 us
// = 4.5 TB/s (25 of 32 lanes have a chunk); the sum of the partials another 5 us.
// FROM8: code 2^e - mean is one fma (code 2^e is exact), with the rounding that x - mean has.
template <typename T, int TPR, int K, int R, bool FROM8, bool STREAM>
__global__ __launch_bounds__(256) void ln_rows_grad_kernel(long long rows, int C, const T* __restrict__ dy, int dys,
                                                           const T* __restrict__ x, int xs,
                                                           const signed char* __restrict__ codes, int pitch,
                                                           const unsigned char* __restrict__ scales,
                                                           const unsigned char* __restrict__ mask,
                                                           const float* __restrict__ w, const float* __restrict__ b,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           int relu, T* __restrict__ dx, int dxs, int dxcols,
                                                           float* __restrict__ part_w, float* __restrict__ part_b,
                                                           size_t part_stride, int row_blocks) {
  constexpr int VEC = traits<T>::VEC;
  constexpr int RPB = 256 / TPR;
  constexpr int COLS = TPR * K * VEC;
  __shared__ float red[4];
  constexpr int OWN = TPR > 64 ? 0 : 4 * COLS, COLUMN = 8 * ACROSS * VEC;        // of a row, a column workgroup
  __shared__ float fold[OWN > COLUMN ? OWN : COLUMN];
  const int t = threadIdx.x % TPR, rg = threadIdx.x / TPR;
  const int G = (C + rv::GROUP - 1) / rv::GROUP, MB = (C + 7) / 8;
  const bool ragged = (C & (VEC - 1)) != 0;
  // one chunk's dy and x (or codes, scales, ReLU bits) -> xh and dz
  auto terms = [&](const rv::u4_any& rd, const rv::u4_any& rx, const unsigned (&cw)[VEC / 4], const unsigned char (&sc)[2],
                   const unsigned char (&mk)[2], int at, int skip, float mu, float rs, bool live, const float (&g)[VEC],
                   const float (&be)[VEC], float (&xh)[VEC], float (&dz)[VEC]) {
    traits<T>::unpack(rd, dz);
    if (!FROM8) traits<T>::unpack(rx, xh);
    const float a = FROM8 ? rv::group_step(sc[0]) : 0.f, a0 = FROM8 && ragged ? rv::group_step(sc[1]) : a;
    unsigned bits = 0xffffffffu;
    if (FROM8 && mask) bits = ((unsigned)mk[0] | (ragged ? (unsigned)mk[1] << 8 : 0u)) >> (at & 7);
    if (FROM8 && !live) bits = 0u;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float xm = FROM8 ? fmaf(rv::code_at(cw, i), i < skip ? a0 : a, -mu) : xh[i] - mu;
      xh[i] = xm * rs;
      if (FROM8) {
        // bit i as a mask of the whole word
        const unsigned on = (unsigned)__builtin_amdgcn_sbfe((int)bits, i, 1);
        dz[i] = __uint_as_float(__float_as_uint(dz[i]) & on);
      } else {
        const bool off_ = relu && fmaf(xh[i], g[i], be[i]) <= 0.f;          // (a NaN passes, as in the forward)
        dz[i] = live && !off_ ? dz[i] : 0.f;
      }
    }
  };
  if ((int)blockIdx.x >= row_blocks) {                 // a column workgroup: dw and db of ACROSS chunks of columns
    constexpr int SLOTS = 256 / ACROSS, FLY = 2;
    const int slot = threadIdx.x / ACROSS;
    const ln::lane_cols<T, TPR, 1> col((blockIdx.x - row_blocks) * ACROSS + threadIdx.x % ACROSS, C);
    float g[1][VEC], be[1][VEC], aw[VEC], ab[VEC];
    col.params(w, 1.f, C, g);
    col.params(b, 0.f, C, be);
#pragma unroll
    for (int i = 0; i < VEC; ++i) { aw[i] = 0.f; ab[i] = 0.f; }
    for (int base = slot; base < rows; base += SLOTS * FLY) {
      rv::u4_any rx[FLY], rd[FLY];
      float mu[FLY], rs[FLY];
      unsigned cw[FLY][VEC / 4];
      unsigned char sc[FLY][2], mk[FLY][2];
#pragma unroll
      for (int r = 0; r < FLY; ++r) {
        const long long row = min(base + r * SLOTS, (int)rows - 1);
        mu[r] = mean[row];
        rs[r] = rstd[row];
        rd[r] = col.template load<false>(dy + row * dys, 0, 0, C);
        if (FROM8) {
          const int c = min(col.c[0], (C - 1) & ~(VEC - 1)), at = col.at[0];
          rv::load_codes(codes + row * pitch + at, cw[r]);
          sc[r][0] = scales[row * G + c / rv::GROUP];
          if (ragged) sc[r][1] = scales[row * G + at / rv::GROUP];
          if (mask) mk[r][0] = mask[row * MB + at / 8];
          if (mask && ragged) mk[r][1] = mask[row * MB + min(at / 8 + 1, MB - 1)];
        } else {
          rx[r] = col.template load<false>(x + row * xs, 0, 0, C);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < FLY; ++r) {
        float xh[VEC], dz[VEC];
        terms(rd[r], rx[r], cw[r], sc[r], mk[r], col.at[0], col.skip[0], mu[r], rs[r], base + r * SLOTS < rows, g[0], be[0], xh,
              dz);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          aw[i] = fmaf(dz[i], xh[i], aw[i]);
          ab[i] += dz[i];
        }
      }
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
      for (int o = ACROSS; o < 64; o <<= 1) {
        aw[i] += __shfl_xor(aw[i], o, 64);
        ab[i] += __shfl_xor(ab[i], o, 64);
      }
      if (lane < ACROSS) {
        fold[((2 * wave) * ACROSS + lane) * VEC + i] = aw[i];
        fold[((2 * wave + 1) * ACROSS + lane) * VEC + i] = ab[i];
      }
    }
    __syncthreads();
    if (threadIdx.x < ACROSS && col.c[0] < C) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (col.own[0][i] != 0.f) {
          float s[2];
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            const float* const f = fold + (which * ACROSS + threadIdx.x) * VEC + i;
            constexpr int W = 2 * ACROSS * VEC;
            s[which] = (f[0] + f[W]) + (f[2 * W] + f[3 * W]);
          }
          part_w[col.at[0] + i] = s[0];
          part_b[col.at[0] + i] = s[1];
        }
    }
    return;
  }
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
  for (long long base = (long long)blockIdx.x * (RPB * R); base < rows; base += (long long)row_blocks * (RPB * R)) {
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
        rd[r][k] = col.template load<STREAM>(db, __umul24(rl, dys), k, C);
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
          rx[r][k] = col.template load<STREAM>(xb, __umul24(rl, xs), k, C);
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
        terms(rd[r][k], rx[r][k], cw[r][k], sc[r][k], mk[r][k], col.at[k], col.skip[k], mu[r], rs[r], live, g[k], be[k], v[k],
              d[k]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = v[k][i], dz = d[k][i];
          aw[k][i] = fmaf(dz, xh, aw[k][i]);
          ab[k][i] += dz;
          // summed here: put off behind the row's sums, the terms stay alive
          asm volatile("" : "+v"(aw[k][i]), "+v"(ab[k][i]));
          const float u = dz * g[k][i], um = u * col.own[k][i];
          s1 += um;
          s2 = fmaf(um, xh, s2);
          d[k][i] = u;
        }
      }
      if (dx) {
        s1 = row_sum<TPR>(s1, red) * rc;
        s2 = row_sum<TPR>(s2, red) * rc;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] = rs[r] * fmaf(-s2, v[k][i], d[k][i] - s1);
          if (live) col.template store<STREAM>(ob, __umul24(rl, dxs), k, C, o);
        }
        if (dxcols > C && live)
#pragma unroll 1
          for (int c = C + t; c < dxcols; c += TPR)
            traits<T>::store1(rv::at32(ob, (__umul24(rl, dxs) + c) * (unsigned)sizeof(T)), 0.f);
      }
    }
  }
  if (!part_w || (int)gridDim.x > row_blocks) return;
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

// Column workgroups of a call.  A call of few rows is one launch: workgroups for dx, and one for every ACROSS chunks of
// columns that goes through all the rows again (by then they are in a cache) for dw and db -- no partial sums, no second
// launch, which costs the host 4 us.  512 x 512: 14 us a call, 18 with two launches; 2048 x 512: 14, 18; 4096 x 256: 19, 18;
// 2048 x 1536: 24, 18.
int rows_grad_columns(int dtype, long long rows, int C) {
  const int wide = ACROSS * ln::vec_of(dtype);
  return rows <= 2048 && rows * C <= 3 << 19 ? (C + wide - 1) / wide : 0;
}

// Workgroups of a rows backward launch = its partial sums: `per` a CU, as many as keep memory busy and no more, each with
// four rows at least where it takes a row at a time.  A CU (dx, dweight, dbias from x / from 8 bits, us; all cached):
//   one chunk a lane   bf16 786432 x 128: 3 118 / 112, 4 120 / 108, 6 131 / 112
//                      fp32 393216 x 128: 3 115 / 95, 4 115 / 92, 8 124 / 101
//   two, a wave a row  bf16 46000 x 753: 2 48 / 51, 3 45 / 48, 4 57 / 57;  fp32 98304 x 512: 2 116 / 91, 3 118 / 92
//   two, a workgroup   bf16 16384 x 4000: 2 90 / 92, 3 98 / 90, 4 124 / 109;  fp32 10000 x 1501: 2 43 / 43, 3 41 / 38
//   four, eight        fp32 8192 x 4096: 1 93 / 80, 2 87 / 70, 4 97 / 81;  bf16 4096 x 8192: 1 67 / 65, 2 81 / 80
int rows_grad_parts(int dtype, long long rows, int C) {
  const int vec = ln::vec_of(dtype), tpr = ln::rows_threads(C, vec), k = (C + tpr * vec - 1) / (tpr * vec);
  const int per = k == 1 ? 4 : k == 2 ? ((vec == 8) == (tpr == 64) ? 3 : 2) : vec == 4 && k <= 4 ? 2 : 1;
  const long long n = tpr == 256 ? (rows + 3) / 4 : ln::rows_blocks(rows, tpr, k == 1 ? 2 : 1);
  return (int)(n < 256 * per ? n : 256 * per);
}

template <typename T>
int rows_backward(int parts, int columns, long long rows, int C, const void* dy, long long dys, const void* x, long long xs,
                  const void* codes, long long pitch, const void* scales, const void* mask, const float* w, const float* b,
                  const float* mean, const float* rstd, int relu, void* dx, long long dxs, int dxcols, float* pw, float* pb,
                  size_t ps, hipStream_t st) {
  const bool stream = rows * C * (long long)sizeof(T) >= rv::STREAM_BYTES;
#define LN_ONE(T, TPR, K, R, FROM8, STREAM)                                                                               \
  hipLaunchKernelGGL((ln_rows_grad_kernel<T, TPR, K, R, FROM8, STREAM>), dim3(parts + columns), dim3(256), 0, st, rows,   \
                     C, (const T*)dy, (int)dys, (const T*)x, (int)xs, (const signed char*)codes, (int)pitch,              \
                     (const unsigned char*)scales, (const unsigned char*)mask, w, b, mean, rstd, relu, (T*)dx, (int)dxs,  \
                     dxcols, pw, pb, ps, parts)
#define LN_CALL(T, TPR, K, R)                                \
  do {                                                       \
    if (codes && stream) LN_ONE(T, TPR, K, R, true, true);   \
    else if (codes) LN_ONE(T, TPR, K, R, true, false);       \
    else if (stream) LN_ONE(T, TPR, K, R, false, true);      \
    else LN_ONE(T, TPR, K, R, false, false);                 \
  } while (0)
  LN_ROWS_PICK(T, C, LN_CALL);
#undef LN_CALL
#undef LN_ONE
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" size_t pvn3d_layer_norm_grad_workspace_bytes(int dtype, long long rows, int C) {
  if (rows <= 0 || C <= 0 || C > ln::MAX_C || dtype < 0 || dtype > 2) return 0;
  if (rows_grad_columns(dtype, rows, C)) return 0;
  return (size_t)rows_grad_parts(dtype, rows, C) * 2 * C * sizeof(float);
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
  if (!codes) scales = mask = nullptr;
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
  const int columns = dweight ? rows_grad_columns(dtype, rows, C) : 0;
  const int parts = dx || !columns ? rows_grad_parts(dtype, rows, C) : 0;
  if (dweight && !columns && (!workspace || workspace_bytes < (size_t)parts * 2 * C * sizeof(float)))
    return (int)hipErrorInvalidValue;
  float* const part = (float*)workspace;
  float* const pw = dweight && !columns ? part : dweight;
  float* const pb = dweight && !columns ? part + C : dbias;
  const auto run = dtype == 0 ? rows_backward<float> : dtype == 1 ? rows_backward<bf16> : rows_backward<fp16>;
  const int rc = run(parts, columns, rows, C, dy, dys, x, xs, codes, pitch, scales, mask, weight, bias, mean, rstd, relu, dx,
                     dxs, dx_cols, pw, pb, 2 * (size_t)C, (hipStream_t)stream);
  if (rc || !dweight || columns) return rc;
  return rv::fold(parts, 2 * (size_t)C, C, part, dweight, dbias, (hipStream_t)stream);
}
