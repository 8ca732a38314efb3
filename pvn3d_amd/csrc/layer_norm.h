// layer_norm.h -- what the layer-norm translation units share: row sums, launch shapes, the sum of the partial gradients.
#pragma once
#include "rowvec.h"

namespace ln {

using rv::bf16;
using rv::fp16;
using rv::traits;

constexpr int MAX_C = 8192;
// Row strides the kernels take: a workgroup addresses its rows (512 at most) as one base and 32-bit byte offsets -- the
// 64-bit products of a row index cost more than the arithmetic on the row.
constexpr long long MAX_STRIDE = 1 << 20;

// sum over the TPR lanes of a row; TPR = 256: over the workgroup (a barrier: every thread of it calls this)
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = rv::lanes_sum<(TPR < 64 ? TPR : 64)>(v);
  if (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// The chunks of one row of a thread, in registers: chunk k's window, and which of its values are this lane's own (1 / 0).
// TPR = 1 is the kernel for C <= VEC: one thread holds the whole row, value by value.
template <typename T, int TPR, int K>
struct lane_cols {
  static constexpr int VEC = traits<T>::VEC;
  int c[K], at[K], skip[K];
  float own[K][VEC];
  __device__ __forceinline__ lane_cols(int t, int C) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      c[k] = (k * TPR + t) * VEC;
      at[k] = 0;
      skip[k] = 0;
      if (TPR > 1) {
        const rv::window<VEC> w(c[k], C);
        at[k] = w.at;
        skip[k] = w.skip;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) own[k][i] = i >= skip[k] && at[k] + i < C ? 1.f : 0.f;
    }
  }
  __device__ __forceinline__ void params(const float* __restrict__ p, float missing, int C, float (&v)[K][VEC]) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        float f[4] = {missing, missing, missing, missing};
        if (TPR == 1) {                                // nothing behind C: a ReLU's bits there are off
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = i + j < C ? p ? p[i + j] : missing : 0.f;
        } else if (p) {
          traits<float>::unpack(*reinterpret_cast<const rv::u4_any*>(p + at[k] + i), f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][i + j] = f[j];
      }
  }
  // the chunk as loaded; row: its place behind base, in elements
  template <bool STREAM>
  __device__ __forceinline__ rv::u4_any load(const T* __restrict__ base, unsigned row, int k, int C) const {
    const T* const p = rv::at32(base, (row + at[k]) * (unsigned)sizeof(T));
    rv::u4_any r;
    if (TPR > 1) {
      rv::get<STREAM>(p, r);
      return r;
    }
    float v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = i < C ? traits<T>::load1(p + i) : 0.f;
    return traits<T>::pack(v);                         // (exact: the values are of type T)
  }
  template <bool STREAM>
  __device__ __forceinline__ void store(T* __restrict__ base, unsigned row, int k, int C, const float (&v)[VEC]) const {
    T* const p = rv::at32(base, (row + at[k]) * (unsigned)sizeof(T));
    if (TPR > 1) {
      if (c[k] < C) rv::store_vec<T, STREAM>(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i < C) traits<T>::store1(p + i, v[i]);
    }
  }
};

inline int vec_of(int dtype) { return dtype == 0 ? 4 : 8; }

// threads per row: the power of two whose chunks cover it, 64 at most with up to two chunks each; beyond that a workgroup
inline int rows_threads(int C, int vec) {
  const int chunks = (C + vec - 1) / vec;
  int t = 1;
  while (t < chunks && t < 64) t <<= 1;
  return chunks > 2 * 64 ? 256 : t;
}
inline long long rows_blocks(long long rows, int tpr, int r) {
  const long long per = (long long)(256 / tpr) * r;
  return (rows + per - 1) / per;
}

// the (threads per row, chunks, rows in flight) instance for C columns
#define LN_ROWS_PICK(T, C, CALL)                                          \
  do {                                                                    \
    constexpr int vec__ = rv::traits<T>::VEC;                             \
    const int tpr__ = ln::rows_threads(C, vec__);                         \
    const int k__ = (C + tpr__ * vec__ - 1) / (tpr__ * vec__);            \
    if (tpr__ == 1) CALL(T, 1, 1, 2);                                     \
    else if (tpr__ == 2) CALL(T, 2, 1, 2);                                \
    else if (tpr__ == 4) CALL(T, 4, 1, 2);                                \
    else if (tpr__ == 8) CALL(T, 8, 1, 2);                                \
    else if (tpr__ == 16) CALL(T, 16, 1, 2);                              \
    else if (tpr__ == 32) CALL(T, 32, 1, 2);                              \
    else if (tpr__ == 64 && k__ == 1) CALL(T, 64, 1, 2);                  \
    else if (tpr__ == 64) CALL(T, 64, 2, 1);                              \
    else if (k__ == 1) CALL(T, 256, 1, 2);                                \
    else if (k__ == 2) CALL(T, 256, 2, 1);                                \
    else if (vec__ == 8 || k__ <= 4) CALL(T, 256, 4, 1);                  \
    else CALL(T, 256, (vec__ == 8 ? 4 : 8), 1);                           \
  } while (0)

}  // namespace ln
