// layer_norm_chan.hip -- layer norm over the channels of (B, C, M) tensors, M contiguous: the layout in which the modules
// hand features on.  The formulas are those of layer_norm.hip.
//
// 16 lanes x 4 consecutive points across, blockDim.x / 16 channel slots down: a thread holds channels cy, cy + CY, ... (KC
// of them) of its four points in registers, as loaded (unpacked at each use), so memory is read once.  The sums over the
// channels go through two shuffles and one LDS exchange; two LDS buffers in turn, one barrier per sum.  KC = 0: more
// channels than the registers of 1024 threads hold -- x is read again for every pass.
#include "layer_norm.h"

namespace {

using rv::bf16;
using rv::fp16;
using rv::traits;

constexpr int PTS = 4;                               // points per thread
constexpr int MAX_THREADS = 1024;

template <typename T> struct raw4 { rv::u2_any r; };
template <> struct raw4<float> { rv::u4_any r; };

template <typename T>
__device__ __forceinline__ void open(const raw4<T>& a, float (&v)[4]) {
  float f[8];
  traits<T>::unpack(rv::u4_any{a.r.x, a.r.y, 0, 0}, f);
  v[0] = f[0]; v[1] = f[1]; v[2] = f[2]; v[3] = f[3];
}
template <>
__device__ __forceinline__ void open<float>(const raw4<float>& a, float (&v)[4]) { traits<float>::unpack(a.r, v); }

template <typename T>
__device__ __forceinline__ raw4<T> shut(const float (&v)[4]) {
  return raw4<T>{rv::u2_any{traits<T>::p2(v[0], v[1]), traits<T>::p2(v[2], v[3])}};
}
template <>
__device__ __forceinline__ raw4<float> shut<float>(const float (&v)[4]) { return raw4<float>{traits<float>::pack(v)}; }

// Chunks are whole and unconditional: the last, partial one of a row of points is taken as its last four points, which
// overlap the neighbour's -- computed and stored twice, with the same bits, and left out of dw and db.
struct tile_at {
  int b, m0, skip;
  bool live;
  __device__ __forceinline__ tile_at(int tile, int NV, int MV, int M) {
    const int pv = tile * 16 + (threadIdx.x & 15);
    live = pv < NV;
    const int at = live ? pv : NV - 1;
    b = at / MV;
    const int m = (at - b * MV) * PTS;
    m0 = min(m, M - PTS);
    skip = m - m0;
  }
};

// s[i] -> sum over the workgroup's channel slots of s[i], for the thread's own points
template <int N>
__device__ __forceinline__ void slot_sum(float (&s)[N], float (*buf)[16 * N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, px = lane & 15, waves = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = rv::add32(rv::add16(s[i]));
  if (lane < 16) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[wave][px * N + i] = s[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = 0.f;
  for (int wv = 0; wv < waves; ++wv)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += buf[wv][px * N + i];
}

template <typename T, int KC>
__global__ __launch_bounds__(MAX_THREADS) void ln_chan_kernel(int B, int C, int M, int MV, const T* __restrict__ x,
                                                              const float* __restrict__ w, const float* __restrict__ b,
                                                              float eps, int relu, T* __restrict__ y,
                                                              float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int KR = KC > 0 ? KC : 1;
  __shared__ float buf[2][MAX_THREADS / 64][16 * PTS];
  const int cy = threadIdx.x >> 4, CY = blockDim.x >> 4;
  const int NV = B * MV;
  const float rc = 1.f / (float)C, floor = relu ? 0.f : -__builtin_inff();
  for (int tile = blockIdx.x; tile < (NV + 15) / 16; tile += gridDim.x) {
    const tile_at at(tile, NV, MV, M);
    const size_t off = (size_t)at.b * C * M + at.m0;
    const T* const p = x + off;
    T* const q = y + off;
    raw4<T> r[KR];
    float s[PTS] = {0.f, 0.f, 0.f, 0.f}, mu[PTS], rs[PTS];
    if (KC > 0) {
#pragma unroll
      for (int k = 0; k < KR; ++k) {
        const int c = cy + k * CY;
        r[k] = *reinterpret_cast<const raw4<T>*>(p + (size_t)(c < C ? c : 0) * M);
      }
    }
    // f(channel, values) for each of the thread's channels
    auto each = [&](auto f) {
      float v[PTS];
      if (KC > 0) {
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          if (cy + k * CY < C) {
            open<T>(r[k], v);
            f(cy + k * CY, v);
          }
        }
      } else {
        for (int c = cy; c < C; c += CY) {
          open<T>(*reinterpret_cast<const raw4<T>*>(p + (size_t)c * M), v);
          f(c, v);
        }
      }
    };
    each([&](int, const float (&v)[PTS]) {
#pragma unroll
      for (int i = 0; i < PTS; ++i) s[i] += v[i];
    });
    slot_sum<PTS>(s, buf[0]);
#pragma unroll
    for (int i = 0; i < PTS; ++i) { mu[i] = s[i] * rc; s[i] = 0.f; }
    each([&](int, const float (&v)[PTS]) {
#pragma unroll
      for (int i = 0; i < PTS; ++i) s[i] = fmaf(v[i] - mu[i], v[i] - mu[i], s[i]);
    });
    slot_sum<PTS>(s, buf[1]);
#pragma unroll
    for (int i = 0; i < PTS; ++i) rs[i] = 1.f / sqrtf(s[i] * rc + eps);
    if (at.live && cy == 0) {
#pragma unroll
      for (int i = 0; i < PTS; ++i) {
        mean[(size_t)at.b * M + at.m0 + i] = mu[i];
        rstd[(size_t)at.b * M + at.m0 + i] = rs[i];
      }
    }
    each([&](int c, const float (&v)[PTS]) {
      const float g = w ? w[c] : 1.f, be = b ? b[c] : 0.f;
      float z[PTS];
#pragma unroll
      for (int i = 0; i < PTS; ++i)                      // (maximum: a NaN stays one)
        z[i] = __builtin_elementwise_maximum(fmaf((v[i] - mu[i]) * rs[i], g, be), floor);
      if (at.live) *reinterpret_cast<raw4<T>*>(q + (size_t)c * M) = shut<T>(z);
    });
  }
}

// dw / db: a thread has the same channels for all its tiles: a register each, summed over the 16 lanes at the end (KC = 0:
// in LDS, summed over the lanes per tile; dynamic LDS, 2 C floats).
template <typename T, int KC>
__global__ __launch_bounds__(MAX_THREADS) void ln_chan_grad_kernel(int B, int C, int M, int MV, const T* __restrict__ dy,
                                                                   const T* __restrict__ x, const float* __restrict__ w,
                                                                   const float* __restrict__ b,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd, int relu,
                                                                   T* __restrict__ dx, float* __restrict__ part) {
  constexpr int KR = KC > 0 ? KC : 1;
  __shared__ float buf[2][MAX_THREADS / 64][16 * 2 * PTS];
  extern __shared__ float lacc[];
  const int px = threadIdx.x & 15, cy = threadIdx.x >> 4, CY = blockDim.x >> 4;
  const int NV = B * MV;
  const float rc = 1.f / (float)C;
  float aw[KR], ab[KR];
#pragma unroll
  for (int k = 0; k < KR; ++k) { aw[k] = 0.f; ab[k] = 0.f; }
  if (KC == 0) {
    for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) lacc[c] = 0.f;
    __syncthreads();
  }
  int turn = 0;
  for (int tile = blockIdx.x; tile < (NV + 15) / 16; tile += gridDim.x, turn ^= 1) {
    const tile_at at(tile, NV, MV, M);
    const size_t off = (size_t)at.b * C * M + at.m0;
    raw4<T> rx[KR], rd[KR];
    float mu[PTS], rs[PTS], s[2 * PTS];
#pragma unroll
    for (int i = 0; i < PTS; ++i) {
      const size_t mi = (size_t)at.b * M + at.m0 + i;
      mu[i] = mean[mi];
      rs[i] = rstd[mi];
      s[i] = 0.f;
      s[PTS + i] = 0.f;
    }
    if (KC > 0) {
#pragma unroll
      for (int k = 0; k < KR; ++k) {
        const size_t o = off + (size_t)(cy + k * CY < C ? cy + k * CY : 0) * M;
        rx[k] = *reinterpret_cast<const raw4<T>*>(x + o);
        rd[k] = *reinterpret_cast<const raw4<T>*>(dy + o);
      }
    }
    // f(k, channel, xh, dz, weight) for each of the thread's channels; dz = 0 where the ReLU is off and in a lane without
    // points
    auto each = [&](auto f) {
      float v[PTS], d[PTS];
      auto one = [&](int k, int c) {
        const float g = w ? w[c] : 1.f, be = b ? b[c] : 0.f;
#pragma unroll
        for (int i = 0; i < PTS; ++i) {
          v[i] = (v[i] - mu[i]) * rs[i];
          const bool off_ = relu && fmaf(v[i], g, be) <= 0.f;      // (a NaN passes, as in the forward)
          d[i] = at.live && !off_ ? d[i] : 0.f;
        }
        f(k, c, v, d, g);
      };
      if (KC > 0) {
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          if (cy + k * CY < C) {
            open<T>(rx[k], v);
            open<T>(rd[k], d);
            one(k, cy + k * CY);
          }
        }
      } else {
        for (int c = cy; c < C; c += CY) {
          open<T>(*reinterpret_cast<const raw4<T>*>(x + off + (size_t)c * M), v);
          open<T>(*reinterpret_cast<const raw4<T>*>(dy + off + (size_t)c * M), d);
          one(0, c);
        }
      }
    };
    each([&](int k, int c, const float (&xh)[PTS], const float (&dz)[PTS], float g) {
      float w1 = 0.f, b1 = 0.f;
#pragma unroll
      for (int i = 0; i < PTS; ++i) {
        const float own = i >= at.skip ? dz[i] : 0.f;
        w1 = fmaf(own, xh[i], w1);
        b1 += own;
        s[i] = fmaf(dz[i], g, s[i]);
        s[PTS + i] = fmaf(dz[i] * g, xh[i], s[PTS + i]);
      }
      if (KC > 0) {
        aw[k] += w1;
        ab[k] += b1;
      } else {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
          w1 += __shfl_xor(w1, o, 64);
          b1 += __shfl_xor(b1, o, 64);
        }
        if (px == 0) {                               // the one thread that adds to this channel's words
          lacc[c] += w1;
          lacc[C + c] += b1;
        }
      }
    });
    if (!dx) continue;
    slot_sum<2 * PTS>(s, buf[turn]);
#pragma unroll
    for (int i = 0; i < 2 * PTS; ++i) s[i] *= rc;
    each([&](int, int c, const float (&xh)[PTS], const float (&dz)[PTS], float g) {
      float o[PTS];
#pragma unroll
      for (int i = 0; i < PTS; ++i) o[i] = rs[i] * (dz[i] * g - s[i] - xh[i] * s[PTS + i]);
      if (at.live) *reinterpret_cast<raw4<T>*>(dx + off + (size_t)c * M) = shut<T>(o);
    });
  }
  if (!part) return;
  float* const pw = part + (size_t)blockIdx.x * 2 * C;
  if (KC > 0) {
#pragma unroll
    for (int k = 0; k < KR; ++k) {
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        aw[k] += __shfl_xor(aw[k], o, 64);
        ab[k] += __shfl_xor(ab[k], o, 64);
      }
      const int c = cy + k * CY;
      if (px == 0 && c < C) {
        pw[c] = aw[k];
        pw[C + c] = ab[k];
      }
    }
  } else {
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) pw[c] = lacc[c];
  }
}

// threads and channels per thread: 16 slots up to 128 channels, then 8 channels a slot up to 512
void chan_shape(int C, int& threads, int& kc) {
  int cy = 16;
  if (C > 128) cy = (C + 31) / 32 * 4;
  if (C > 512) cy = 64;
  threads = cy * 16;
  const int k = (C + cy - 1) / cy;
  kc = k <= 1 ? 1 : k <= 2 ? 2 : k <= 4 ? 4 : k <= 8 ? 8 : 0;
}
int points4(int M) { return (int)(((long long)M + PTS - 1) / PTS); }
long long chan_tiles(int B, int M) { return ((long long)B * points4(M) + 15) / 16; }
int chan_grad_parts(int B, int M) {
  const long long n = chan_tiles(B, M);
  return (int)(n < ln::MAX_PARTS ? n : ln::MAX_PARTS);
}
bool chan_ok(int dtype, int B, int C, int M) {
  return dtype >= 0 && dtype <= 2 && C > 0 && C <= ln::MAX_C && B >= 0 && (M == 0 || M >= PTS) && (long long)B * points4(M) < 0x7fffff00LL;
}

template <typename T>
int chan_forward(int B, int C, int M, const void* x, const float* w, const float* b, float eps, int relu, void* y,
                 float* mean, float* rstd, hipStream_t st) {
  int threads, kc;
  chan_shape(C, threads, kc);
  const long long tiles = chan_tiles(B, M);
  const dim3 grid((unsigned)(tiles < 16384 ? tiles : 16384));
#define LN_CALL(KC)                                                                                              \
  hipLaunchKernelGGL((ln_chan_kernel<T, KC>), grid, dim3(threads), 0, st, B, C, M, points4(M), (const T*)x, w, b, \
                     eps, relu, (T*)y, mean, rstd)
  switch (kc) {
    case 1: LN_CALL(1); break;
    case 2: LN_CALL(2); break;
    case 4: LN_CALL(4); break;
    case 8: LN_CALL(8); break;
    default: LN_CALL(0); break;
  }
#undef LN_CALL
  PVN3D_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int chan_backward(int parts, int B, int C, int M, const void* dy, const void* x, const float* w, const float* b,
                  const float* mean, const float* rstd, int relu, void* dx, float* part, hipStream_t st) {
  int threads, kc;
  chan_shape(C, threads, kc);
#define LN_CALL(KC, LDS)                                                                                             \
  hipLaunchKernelGGL((ln_chan_grad_kernel<T, KC>), dim3(parts), dim3(threads), LDS, st, B, C, M, points4(M),        \
                     (const T*)dy, (const T*)x, w, b, mean, rstd, relu, (T*)dx, part)
  switch (kc) {
    case 1: LN_CALL(1, 0); break;
    case 2: LN_CALL(2, 0); break;
    case 4: LN_CALL(4, 0); break;
    case 8: LN_CALL(8, 0); break;
    default: {
      const int rc = pvn3d_allow_big_lds(ln_chan_grad_kernel<T, 0>);
      if (rc) return rc;
      LN_CALL(0, 2 * C * sizeof(float));
    }
  }
#undef LN_CALL
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" size_t pvn3d_layer_norm_chan_grad_workspace_bytes(int dtype, int B, int C, int M) {
  if (!chan_ok(dtype, B, C, M)) return 0;
  return (size_t)chan_grad_parts(B, M) * 2 * C * sizeof(float);
}

extern "C" int pvn3d_layer_norm_chan(int dtype, int B, int C, int M, const void* x, const float* weight, const float* bias,
                                     float eps, int relu, void* y, float* mean, float* rstd, void* stream) {
  if (!chan_ok(dtype, B, C, M)) return (int)hipErrorInvalidValue;
  if (B == 0 || M == 0) return 0;
  if (!x || !y || !mean || !rstd) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case 0: return chan_forward<float>(B, C, M, x, weight, bias, eps, relu, y, mean, rstd, st);
    case 1: return chan_forward<bf16>(B, C, M, x, weight, bias, eps, relu, y, mean, rstd, st);
    default: return chan_forward<fp16>(B, C, M, x, weight, bias, eps, relu, y, mean, rstd, st);
  }
}

extern "C" int pvn3d_layer_norm_chan_grad(int dtype, int B, int C, int M, const void* dy, const void* x,
                                          const float* weight, const float* bias, const float* mean, const float* rstd,
                                          int relu, void* dx, float* dweight, float* dbias, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (!chan_ok(dtype, B, C, M) || (dweight == nullptr) != (dbias == nullptr) || (!dx && !dweight))
    return (int)hipErrorInvalidValue;
  if (B == 0 || M == 0) {
    if (dweight) {
      pvn3d_fill_u32(dweight, 0, C, st);
      pvn3d_fill_u32(dbias, 0, C, st);
      PVN3D_LAUNCH_CHECK();
    }
    return 0;
  }
  if (!dy || !x || !mean || !rstd) return (int)hipErrorInvalidValue;
  const int parts = chan_grad_parts(B, M);
  if (dweight && (!workspace || workspace_bytes < (size_t)parts * 2 * C * sizeof(float))) return (int)hipErrorInvalidValue;
  float* part = dweight ? (float*)workspace : nullptr;
  int rc;
  switch (dtype) {
    case 0: rc = chan_backward<float>(parts, B, C, M, dy, x, weight, bias, mean, rstd, relu, dx, part, st); break;
    case 1: rc = chan_backward<bf16>(parts, B, C, M, dy, x, weight, bias, mean, rstd, relu, dx, part, st); break;
    default: rc = chan_backward<fp16>(parts, B, C, M, dy, x, weight, bias, mean, rstd, relu, dx, part, st); break;
  }
  if (rc || !dweight) return rc;
  return rv::fold(parts, 2 * (size_t)C, C, part, dweight, dbias, st);
}
