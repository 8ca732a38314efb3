// layer_norm_chan.hip -- layer norm over the channels of (B, C, M) tensors, M contiguous: the layout in which the modules
// hand features on.  The formulas are those of layer_norm.hip.
//
// A tile is 64 (32, 16) consecutive points of one cloud: PX = 16 (8, 4) lanes x 4 points across, blockDim.x / PX channel
// slots down.  A thread holds channels cy, cy + CY, ... (KC of them) of its four points in registers, as loaded (unpacked at
// each use), so memory is read once.  All addresses are a base that the workgroup shares plus one 32-bit offset per lane (64-bit addresses for
// every channel were half of the registers).  The sums over the channels go through two lane exchanges and one LDS
// exchange; two LDS buffers in turn, one barrier per sum.  KC = 0: more channels than the registers of 1024 threads hold
// -- x is read again for every pass.
// Bound by HBM.  fp32 24 x 128 x 12288 forward 56 us = 5.4 TB/s; bf16 8 x 196 x 16384 backward 38 us = 4.0 TB/s (two
// workgroups a CU load, add up and store in turn).
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

// The compiler forgets what it has derived from a chunk: values unpacked before a barrier are not kept in registers for
// their second use behind it (they were twice the chunk's size).
template <typename T>
__device__ __forceinline__ void forget(raw4<T>& a) {
  unsigned p = a.r.x, q = a.r.y;
  asm volatile("" : "+v"(p), "+v"(q));
  a.r.x = p;
  a.r.y = q;
}
template <>
__device__ __forceinline__ void forget<float>(raw4<float>& a) {
  unsigned p = a.r.x, q = a.r.y, s = a.r.z, t = a.r.w;
  asm volatile("" : "+v"(p), "+v"(q), "+v"(s), "+v"(t));
  a.r = rv::u4_any{p, q, s, t};
}

// Chunks are whole and unconditional: the last, partial one of a row of points is taken as its last four points, which
// overlap the neighbour's -- computed and stored twice, with the same bits, and left out of dw and db.  Lanes behind the
// cloud's last point repeat its last four without a store.
// Tiles of a workgroup.  In turn, or in runs: workgroups are dealt to the eight XCDs in turn, each with an L2 of its own, and
// where neighbouring tiles share memory lines each XCD walks a run of an eighth of the tiles with all its workgroups.
struct tile_walk {
  int at, step, end;
  __device__ __forceinline__ tile_walk(int tiles, int runs, int g) {
    const int b = blockIdx.x;
    if (!runs) {
      at = b;
      step = g;
      end = tiles;
    } else {
      const int per = (tiles + 7) >> 3, x = b & 7;
      at = x * per + (b >> 3);
      step = g >> 3;
      end = min(tiles, (x + 1) * per);
    }
  }
};

template <int PX>
struct tile_at {
  int b, m0, skip;
  bool live;
  __device__ __forceinline__ tile_at(int tile, int per_cloud, int M) {
    b = tile / per_cloud;
    const int m = ((tile - b * per_cloud) * PX + (threadIdx.x & (PX - 1))) * PTS;
    live = m < M;
    m0 = min(m, M - PTS);
    skip = m - m0;
  }
};

// s[i] -> sum over the workgroup's channel slots of s[i], for the thread's own points
template <int N, int PX>
__device__ __forceinline__ void slot_sum(float (&s)[N], float (*buf)[PX * N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, px = lane & (PX - 1), waves = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (PX <= 8) s[i] += __uint_as_float(rv::turn8(__float_as_uint(s[i])));
    if (PX == 4) s[i] += __uint_as_float(rv::turn4(__float_as_uint(s[i])));
    s[i] = rv::add32(rv::add16(s[i]));
  }
  if (lane < PX) {
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

template <typename T, int KC, int PX, bool STREAM>
__global__ __launch_bounds__(MAX_THREADS) void ln_chan_kernel(int tiles, int runs, int per_cloud, int C, int M,
                                                              const T* __restrict__ x,
                                                              const float* __restrict__ w, const float* __restrict__ b,
                                                              float eps, int relu, T* __restrict__ y,
                                                              float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int KR = KC > 0 ? KC : 1;
  __shared__ float buf[2][MAX_THREADS / 64][PX * PTS];
  const int cy = threadIdx.x / PX, CY = blockDim.x / PX;
  const size_t M_ = M, cloud = C * M_, slots = (size_t)CY * M;      // slots: elements between a thread's channels
  const float rc = 1.f / (float)C;
  float low = relu ? 0.f : -__builtin_inff();
  asm("" : "+v"(low));             // a register, not a choice of two constants at every use
  float gk[KR], bk[KR];
  bool has[KR];                    // (only the last of a thread's channels can be missing)
#pragma unroll
  for (int k = 0; k < KR; ++k) {
    const int c = cy + k * CY;
    has[k] = k < KR - 1 || c < C;
    gk[k] = KC > 0 && w && has[k] ? w[c] : 1.f;
    bk[k] = KC > 0 && b && has[k] ? b[c] : 0.f;
  }
  const int clast = KC > 0 ? min(cy, C - 1 - (KR - 1) * CY) : 0;
  const tile_walk walk(tiles, runs, gridDim.x);
  for (int tile = walk.at; tile < walk.end; tile += walk.step) {
    const tile_at<PX> at(tile, per_cloud, M);
    const T* const p = x + at.b * cloud;
    T* const q = y + at.b * cloud;
    const unsigned o = (unsigned)(cy * M + at.m0) * (unsigned)sizeof(T);
    const unsigned ol = (unsigned)(clast * M + at.m0) * (unsigned)sizeof(T);
    raw4<T> r[KR];
    float s[PTS] = {0.f, 0.f, 0.f, 0.f}, mu[PTS], rs[PTS];
    if (KC > 0) {
#pragma unroll
      for (int k = 0; k < KR; ++k) rv::get<STREAM>(rv::at32(p + k * slots, k < KR - 1 ? o : ol), r[k].r);
      __builtin_amdgcn_sched_barrier(0);     // all loads on their way before anything waits for one
    }
    // f(k, channel's base, channel, values) for each of the thread's channels
    auto each = [&](auto f) {
      float v[PTS];
      if (KC > 0) {
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          if (has[k]) {
            open<T>(r[k], v);
            f(k, k * slots, cy + k * CY, v);
          }
        }
      } else {
        size_t at_c = 0;
        for (int c = cy; c < C; c += CY, at_c += slots) {
          open<T>(*reinterpret_cast<const raw4<T>*>(rv::at32(p + at_c, o)), v);
          f(0, at_c, c, v);
        }
      }
    };
    each([&](int, size_t, int, const float (&v)[PTS]) {
#pragma unroll
      for (int i = 0; i < PTS; ++i) s[i] += v[i];
    });
    slot_sum<PTS, PX>(s, buf[0]);
#pragma unroll
    for (int i = 0; i < PTS; ++i) { mu[i] = s[i] * rc; s[i] = 0.f; }
    each([&](int, size_t, int, const float (&v)[PTS]) {
#pragma unroll
      for (int i = 0; i < PTS; ++i) s[i] = fmaf(v[i] - mu[i], v[i] - mu[i], s[i]);
    });
    slot_sum<PTS, PX>(s, buf[1]);
#pragma unroll
    for (int i = 0; i < PTS; ++i) rs[i] = __builtin_amdgcn_rsqf(fmaf(s[i], rc, eps));       // v_rsq_f32: within one ulp
    if (at.live && cy == 0) {
#pragma unroll
      for (int i = 0; i < PTS; ++i) {
        mean[at.b * M_ + at.m0 + i] = mu[i];
        rstd[at.b * M_ + at.m0 + i] = rs[i];
      }
    }
    each([&](int k, size_t at_c, int c, const float (&v)[PTS]) {
      const float g = KC > 0 ? gk[k] : w ? w[c] : 1.f, be = KC > 0 ? bk[k] : b ? b[c] : 0.f;
      float z[PTS];
#pragma unroll
      for (int i = 0; i < PTS; ++i)                      // (maximum: a NaN stays one)
        z[i] = __builtin_elementwise_maximum(fmaf((v[i] - mu[i]) * rs[i], g, be), low);
      if (at.live) rv::put<STREAM>(rv::at32(q + at_c, o), shut<T>(z).r);
    });
  }
}

// dw / db: a thread has the same channels for all its tiles: a register each, summed over the 16 lanes at the end (KC = 0:
// in LDS, summed over the lanes per tile; dynamic LDS, 2 C floats).
// CHANNELS: the call has channel workgroups (an instance of its own: they take registers).
template <typename T, int KC, int PX, bool CHANNELS, bool STREAM>
__global__ __launch_bounds__(MAX_THREADS) void ln_chan_grad_kernel(int tiles, int runs, int per_cloud, int C, int M,
                                                                   const T* __restrict__ dy, const T* __restrict__ x,
                                                                   const float* __restrict__ w, const float* __restrict__ b,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd, int relu,
                                                                   T* __restrict__ dx, float* __restrict__ part_w,
                                                                   float* __restrict__ part_b, size_t part_stride,
                                                                   int tile_blocks) {
  if (CHANNELS && (int)blockIdx.x >= tile_blocks) {       // a channel workgroup: a wave for dw and db of a channel
    const int lane = threadIdx.x & 63, c = ((blockIdx.x - tile_blocks) * blockDim.x + threadIdx.x) >> 6;
    if (c >= C) return;
    const float g = w ? w[c] : 1.f, be = b ? b[c] : 0.f;
    const int per = (M + PTS - 1) / PTS, clouds = tiles / per_cloud, chunks = clouds * per;
    float w1 = 0.f, b1 = 0.f;
    for (int base = lane; base < chunks; base += 2 * 64) {
      raw4<T> rx[2], rd[2];
      rv::u4_any mu_[2], rs_[2];
      int skip[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int q = min(base + r * 64, chunks - 1), cl = q / per, m = (q - cl * per) * PTS, m0 = min(m, M - PTS);
        const size_t at = ((size_t)cl * C + c) * M + m0, point = (size_t)cl * M + m0;
        skip[r] = base + r * 64 < chunks ? m - m0 : PTS;
        rx[r] = *reinterpret_cast<const raw4<T>*>(x + at);
        rd[r] = *reinterpret_cast<const raw4<T>*>(dy + at);
        mu_[r] = *reinterpret_cast<const rv::u4_any*>(mean + point);
        rs_[r] = *reinterpret_cast<const rv::u4_any*>(rstd + point);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v[PTS], d[PTS], mu[PTS], rs[PTS];
        open<T>(rx[r], v);
        open<T>(rd[r], d);
        traits<float>::unpack(mu_[r], mu);
        traits<float>::unpack(rs_[r], rs);
#pragma unroll
        for (int i = 0; i < PTS; ++i) {
          const float xh = (v[i] - mu[i]) * rs[i];
          const bool off_ = relu && fmaf(xh, g, be) <= 0.f;
          const float dz = i >= skip[r] && !off_ ? d[i] : 0.f;
          w1 = fmaf(dz, xh, w1);
          b1 += dz;
        }
      }
    }
    w1 = rv::lanes_sum<64>(w1);
    b1 = rv::lanes_sum<64>(b1);
    if (lane == 0) {
      part_w[c] = w1;
      part_b[c] = b1;
    }
    return;
  }
  constexpr int KR = KC > 0 ? KC : 1;
  __shared__ float buf[2][MAX_THREADS / 64][PX * 2 * PTS];
  extern __shared__ float lacc[];
  const int px = threadIdx.x & (PX - 1), cy = threadIdx.x / PX, CY = blockDim.x / PX;
  const size_t M_ = M, cloud = C * M_, slots = (size_t)CY * M;      // slots: elements between a thread's channels
  const float rc = 1.f / (float)C;
  float aw[KR], ab[KR], gk[KR], bk[KR];
  bool has[KR];                    // (only the last of a thread's channels can be missing)
#pragma unroll
  for (int k = 0; k < KR; ++k) {
    const int c = cy + k * CY;
    has[k] = k < KR - 1 || c < C;
    aw[k] = 0.f;
    ab[k] = 0.f;
    gk[k] = KC > 0 && w && has[k] ? w[c] : 1.f;
    bk[k] = KC > 0 && b && has[k] ? b[c] : 0.f;
  }
  const int clast = KC > 0 ? min(cy, C - 1 - (KR - 1) * CY) : 0;
  if (KC == 0) {
    for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) lacc[c] = 0.f;
    __syncthreads();
  }
  int turn = 0;
  const tile_walk walk(tiles, runs, tile_blocks);
  for (int tile = walk.at; tile < walk.end; tile += walk.step, turn ^= 1) {
    const tile_at<PX> at(tile, per_cloud, M);
    const T* const px_ = x + at.b * cloud;
    const T* const pd_ = dy + at.b * cloud;
    T* const po_ = dx + at.b * cloud;
    const unsigned o = (unsigned)(cy * M + at.m0) * (unsigned)sizeof(T);
    const unsigned ol = (unsigned)(clast * M + at.m0) * (unsigned)sizeof(T);
    raw4<T> rx[KR], rd[KR];
    float mu[PTS], rs[PTS], s[2 * PTS];
#pragma unroll
    for (int i = 0; i < PTS; ++i) {
      mu[i] = mean[at.b * M_ + at.m0 + i];
      rs[i] = rstd[at.b * M_ + at.m0 + i];
      s[i] = 0.f;
      s[PTS + i] = 0.f;
    }
    if (KC > 0) {
#pragma unroll
      for (int k = 0; k < KR; ++k) {
        rv::get<STREAM>(rv::at32(px_ + k * slots, k < KR - 1 ? o : ol), rx[k].r);
        rv::get<STREAM>(rv::at32(pd_ + k * slots, k < KR - 1 ? o : ol), rd[k].r);
      }
      __builtin_amdgcn_sched_barrier(0);     // all loads on their way before anything waits for one
    }
    // one channel's x, dy -> xh and dz, dz = 0 where the ReLU is off and in a lane without points
    auto one = [&](float g, float be, float (&v)[PTS], float (&d)[PTS]) {
#pragma unroll
      for (int i = 0; i < PTS; ++i) {
        v[i] = (v[i] - mu[i]) * rs[i];
        const bool off_ = relu && fmaf(v[i], g, be) <= 0.f;        // (a NaN passes, as in the forward)
        d[i] = at.live && !off_ ? d[i] : 0.f;
      }
    };
    // its share of the sums over the channels, and of dw, db
    auto add = [&](float g, const float (&xh)[PTS], const float (&dz)[PTS], float& w1, float& b1) {
#pragma unroll
      for (int i = 0; i < PTS; ++i) {
        const float own = i >= at.skip ? dz[i] : 0.f, u = dz[i] * g;
        w1 = fmaf(own, xh[i], w1);
        b1 += own;
        s[i] += u;
        s[PTS + i] = fmaf(u, xh[i], s[PTS + i]);
      }
    };
    // dx = rstd (u - s1 / C - xh s2 / C), from x: xh s2 = (x - mean) (rstd s2) -- rstd^2 would leave fp32's range long before
    // any of these factors does
    auto out = [&](size_t at_c, float g, const float (&v)[PTS], const float (&dz)[PTS]) {
      float e[PTS];
#pragma unroll
      for (int i = 0; i < PTS; ++i) e[i] = rs[i] * fmaf(v[i] - mu[i], s[PTS + i], fmaf(dz[i], g, s[i]));
      if (at.live) rv::put<STREAM>(rv::at32(po_ + at_c, o), shut<T>(e).r);
    };
    float v[PTS], d[PTS];
    if (KC > 0) {
#pragma unroll
      for (int k = 0; k < KR; ++k) {
        if (has[k]) {
          open<T>(rx[k], v);
          open<T>(rd[k], d);
          one(gk[k], bk[k], v, d);
          rd[k] = shut<T>(d);                          // dy with the ReLU's zeros: the same values, exact
          add(gk[k], v, d, aw[k], ab[k]);
          asm volatile("" : "+v"(aw[k]), "+v"(ab[k]));     // summed here: put off behind the barrier, the terms stay alive
          forget<T>(rx[k]);
          forget<T>(rd[k]);
          __builtin_amdgcn_sched_barrier(0);         // one channel after the other
        }
      }
    } else {
      size_t at_c = 0;
      for (int c = cy; c < C; c += CY, at_c += slots) {
        float w1 = 0.f, b1 = 0.f;
        open<T>(*reinterpret_cast<const raw4<T>*>(rv::at32(px_ + at_c, o)), v);
        open<T>(*reinterpret_cast<const raw4<T>*>(rv::at32(pd_ + at_c, o)), d);
        one(w ? w[c] : 1.f, b ? b[c] : 0.f, v, d);
        add(w ? w[c] : 1.f, v, d, w1, b1);
        w1 = rv::lanes_sum<PX>(w1);
        b1 = rv::lanes_sum<PX>(b1);
        if (px == 0) {                                 // the one thread that adds to this channel's words
          lacc[c] += w1;
          lacc[C + c] += b1;
        }
      }
    }
    if (!dx) continue;
    slot_sum<2 * PTS, PX>(s, buf[turn]);
#pragma unroll
    for (int i = 0; i < PTS; ++i) {
      s[i] *= -rc;
      s[PTS + i] *= -rc * rs[i];
    }
    if (KC > 0) {
#pragma unroll
      for (int k = 0; k < KR; ++k) {
        if (has[k]) {
          open<T>(rx[k], v);
          open<T>(rd[k], d);
          out(k * slots, gk[k], v, d);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      size_t at_c = 0;
      for (int c = cy; c < C; c += CY, at_c += slots) {
        const float g = w ? w[c] : 1.f;
        float t[PTS];
        open<T>(*reinterpret_cast<const raw4<T>*>(rv::at32(px_ + at_c, o)), v);
        open<T>(*reinterpret_cast<const raw4<T>*>(rv::at32(pd_ + at_c, o)), d);
#pragma unroll
        for (int i = 0; i < PTS; ++i) t[i] = v[i];
        one(g, b ? b[c] : 0.f, t, d);
        out(at_c, g, v, d);
      }
    }
  }
  if (CHANNELS || !part_w) return;
  float* const pw = part_w + blockIdx.x * part_stride;
  float* const pb = part_b + blockIdx.x * part_stride;
  if (KC > 0) {
#pragma unroll
    for (int k = 0; k < KR; ++k) {
      aw[k] = rv::lanes_sum<PX>(aw[k]);
      ab[k] = rv::lanes_sum<PX>(ab[k]);
      const int c = cy + k * CY;
      if (px == 0 && has[k]) {
        pw[c] = aw[k];
        pb[c] = ab[k];
      }
    }
  } else {
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
      pw[c] = lacc[c];
      pb[c] = lacc[C + c];
    }
  }
}

constexpr int MAX_HELD = 2048;             // channels that the registers of a workgroup hold
// lanes across, threads and channels per thread: 16 lanes and 16 channel slots up to 128 channels, then eight channels a
// slot (8 x 196 x 16384 in bf16, backward: 39.5 us; with six channels a slot and more slots 51.4, with four 52.9); from 257
// channels 8 lanes, so that two workgroups of them still share a CU, from 1025 4 (8 x 1536 x 2048 in bf16: forward 25 us,
// backward 63; 42 and 65 with x read again for every pass, which is left for more than 2048)
struct chan_plan { int px, threads, kc; };
chan_plan chan_shape(int C) {
  chan_plan p;
  p.px = C > MAX_HELD ? 16 : C > 1024 ? 4 : C > 256 ? 8 : 16;
  int cy = 16;
  if (p.px == 4) cy = (C + 127) / 128 * 16;
  else if (p.px == 8) cy = (C + 63) / 64 * 8;
  else if (C > MAX_HELD) cy = 64;
  else if (C > 128) cy = (C + 31) / 32 * 4;
  p.threads = cy * p.px;
  p.kc = C > MAX_HELD ? 0 : (C + cy - 1) / cy;
  return p;
}
int cloud_tiles(int C, int M) { return (int)(((long long)M + chan_shape(C).px * PTS - 1) / (chan_shape(C).px * PTS)); }
long long chan_tiles(int B, int C, int M) { return (long long)B * cloud_tiles(C, M); }
// Whether neighbouring tiles share lines of `line` bytes: their rows start or end within one (23 x 313 x 2324 in bf16: forward
// 30.7 us in turn, 19.7 in runs; backward 50.9, 36.5).  Where they do not, runs are the slower, 24 x 64 x 65536 backward 143 us
// against 133 -- except for the forward and tiles of 128 bytes (24 x 256 x 12288 in bf16 67.4 us, 62.4), so it asks for 256.
bool chan_runs(int elem, int C, int M, int line, long long grid) {
  const long long tile = (long long)chan_shape(C).px * PTS * elem;
  return (grid & 7) == 0 && (tile % line != 0 || (long long)M * elem % line != 0);
}
// Workgroups of a backward launch (every one starts with the parameters and ends with its partial sums): `per` a CU, the
// fewer the more a thread holds.  Backward, a CU: bf16 24 x 128 x 12288: 1 81 us, 2 53, 4 56, 8 59; 24 x 160 x 6000: 2 38,
// 3 61; 24 x 64 x 65536: 2 147, 4 135, 8 151; 24 x 32 x 65536: 4 86, 8 70; fp32 24 x 128 x 12288: 2 102, 4 105, 8 108;
// 24 x 32 x 65536: 2 123, 4 127, 8 136; 24 x 8 x 100000: 4 81, 8 58.
int chan_grad_parts(int dtype, int B, int C, int M) {
  const chan_plan p = chan_shape(C);
  const int few = (dtype == 0 ? 8 : 16) / (p.kc ? p.kc : 1);
  const int per = p.threads > 512 ? 1 : few < 2 ? 2 : few > 8 ? 8 : few;
  const long long n = chan_tiles(B, C, M), most = 256 * per;
  return (int)(n < 8 ? n : n < most ? (n + 7) / 8 * 8 : most);
}
// Channel workgroups of a backward call: as for rows (layer_norm_grad.hip), a call of few points is one launch, with a wave
// for every channel that goes through its points again for dw and db (4 x 64 x 500: 15 us a call, 19 with two launches;
// 1 x 256 x 8192: 15.5, 19; 1 x 512 x 8192: 19, 19; 1 x 64 x 16384: 24, 19).
int chan_grad_channels(int B, int C, int M) {
  const long long points = (long long)B * M;
  const int waves = chan_shape(C).threads / 64;
  return points <= 8192 && points * C <= 1 << 21 ? (C + waves - 1) / waves : 0;
}
constexpr int MAX_POINTS = 1 << 22;        // per cloud: 256 channel slots (chan_shape) of them are within 32-bit byte offsets
bool chan_ok(int dtype, int B, int C, int M) {
  return dtype >= 0 && dtype <= 2 && C > 0 && C <= ln::MAX_C && B >= 0 && (M == 0 || (M >= PTS && M <= MAX_POINTS)) &&
         chan_tiles(B, C, M) < 0x7fffffffLL - 16384;
}

// (8 lanes: seven or eight channels a slot come of 257 to 1024 channels; 4 lanes: eight)
#define LN_CHAN_PICK(CALL)                          \
  if (p.px == 4) {                                  \
    CALL(8, 4);                                     \
  } else if (p.px == 8) {                           \
    if (p.kc <= 7) CALL(7, 8);                      \
    else CALL(8, 8);                                \
  } else {                                          \
    switch (p.kc) {                                 \
      case 1: CALL(1, 16); break;                   \
      case 2: CALL(2, 16); break;                   \
      case 3: CALL(3, 16); break;                   \
      case 4: CALL(4, 16); break;                   \
      case 5: CALL(5, 16); break;                   \
      case 6: CALL(6, 16); break;                   \
      case 7: CALL(7, 16); break;                   \
      case 8: CALL(8, 16); break;                   \
      default: CALL(0, 16); break;                  \
    }                                               \
  }

template <typename T>
int chan_forward(int B, int C, int M, const void* x, const float* w, const float* b, float eps, int relu, void* y,
                 float* mean, float* rstd, hipStream_t st) {
  const chan_plan p = chan_shape(C);
  const long long tiles = chan_tiles(B, C, M);
  // (bf16 24 x 64 x 65536: 84 us, 91 with 8192, 106 with 512; 24 x 32 x 65536: 42, 40, 88, and 45 with one per tile)
  const dim3 grid((unsigned)(tiles < 8 ? tiles : tiles < 16384 ? (tiles + 7) / 8 * 8 : 16384));
  const bool stream = (long long)B * C * M * (long long)sizeof(T) >= rv::STREAM_BYTES;
#define LN_ONE(KC, PX, STREAM)                                                                                              \
  hipLaunchKernelGGL((ln_chan_kernel<T, KC, PX, STREAM>), grid, dim3(p.threads), 0, st, (int)tiles,                         \
                     (int)chan_runs(sizeof(T), C, M, 256, grid.x), cloud_tiles(C, M), C, M,                                 \
                     (const T*)x, w, b, eps, relu, (T*)y, mean, rstd)
#define LN_CALL(KC, PX)                \
  do {                                 \
    if (stream) LN_ONE(KC, PX, true);  \
    else LN_ONE(KC, PX, false);        \
  } while (0)
  LN_CHAN_PICK(LN_CALL)
#undef LN_CALL
#undef LN_ONE
  PVN3D_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int chan_backward(int parts, int channels, int B, int C, int M, const void* dy, const void* x, const float* w, const float* b,
                  const float* mean, const float* rstd, int relu, void* dx, float* pw, float* pb, size_t ps, hipStream_t st) {
  const chan_plan p = chan_shape(C);
  const bool stream = (long long)B * C * M * (long long)sizeof(T) >= rv::STREAM_BYTES;
  const int lds = p.kc ? 0 : (int)(2 * C * sizeof(float));
  if (!p.kc) {
    const int rc = channels ? pvn3d_allow_big_lds(ln_chan_grad_kernel<T, 0, 16, true, false>)
                   : stream ? pvn3d_allow_big_lds(ln_chan_grad_kernel<T, 0, 16, false, true>)
                            : pvn3d_allow_big_lds(ln_chan_grad_kernel<T, 0, 16, false, false>);
    if (rc) return rc;
  }
#define LN_ONE(KC, PX, CHANNELS, STREAM)                                                                                    \
  hipLaunchKernelGGL((ln_chan_grad_kernel<T, KC, PX, CHANNELS, STREAM>), dim3(parts + channels), dim3(p.threads), lds, st,  \
                     (int)chan_tiles(B, C, M), (int)chan_runs(sizeof(T), C, M, 128, parts), cloud_tiles(C, M), C, M,        \
                     (const T*)dy, (const T*)x, w, b, mean, rstd, relu, (T*)dx, pw, pb, ps, parts)
#define LN_CALL(KC, PX)                             \
  do {                                              \
    if (channels) LN_ONE(KC, PX, true, false);      \
    else if (stream) LN_ONE(KC, PX, false, true);   \
    else LN_ONE(KC, PX, false, false);              \
  } while (0)
  LN_CHAN_PICK(LN_CALL)
#undef LN_CALL
#undef LN_ONE
  PVN3D_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" size_t pvn3d_layer_norm_chan_grad_workspace_bytes(int dtype, int B, int C, int M) {
  if (!chan_ok(dtype, B, C, M) || B == 0 || M == 0) return 0;
  return chan_grad_channels(B, C, M) ? 0 : (size_t)chan_grad_parts(dtype, B, C, M) * 2 * C * sizeof(float);
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
  const int channels = dweight ? chan_grad_channels(B, C, M) : 0;
  const int parts = dx || !channels ? chan_grad_parts(dtype, B, C, M) : 0;
  if (dweight && !channels && (!workspace || workspace_bytes < (size_t)parts * 2 * C * sizeof(float)))
    return (int)hipErrorInvalidValue;
  float* const part = (float*)workspace;
  float* const pw = dweight && !channels ? part : dweight;
  float* const pb = dweight && !channels ? part + C : dbias;
  const auto run = dtype == 0 ? chan_backward<float> : dtype == 1 ? chan_backward<bf16> : chan_backward<fp16>;
  const int rc = run(parts, channels, B, C, M, dy, x, weight, bias, mean, rstd, relu, dx, pw, pb, 2 * (size_t)C, st);
  if (rc || !dweight || channels) return rc;
  return rv::fold(parts, 2 * (size_t)C, C, part, dweight, dbias, st);
}
