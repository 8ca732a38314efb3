// layer_norm.h -- what the layer-norm translation units share: row sums, launch shapes, the sum of the partial gradients.
#pragma once
#include "rowvec.h"

namespace ln {

using rv::bf16;
using rv::fp16;
using rv::traits;

constexpr int MAX_C = 8192;
constexpr int MAX_PARTS = 1024;      // workgroups of a backward launch, each with a partial dw and db

// sum over the TPR lanes of a row; TPR = 256: over the workgroup (a barrier: every thread of it calls this)
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) v += __shfl_xor(v, o, 64);
  if (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

inline int vec_of(int dtype) { return dtype == 0 ? 4 : 8; }

// threads per row: the power of two whose chunks cover it, 64 at most; a workgroup where four chunks a lane do not
inline int rows_threads(int cover, int vec) {
  const int chunks = (cover + vec - 1) / vec;
  int t = 1;
  while (t < chunks && t < 64) t <<= 1;
  return chunks > 4 * 64 ? 256 : t;
}
inline long long rows_blocks(long long rows, int tpr, int r) {
  const long long per = (long long)(256 / tpr) * r;
  return (rows + per - 1) / per;
}

// the (threads per row, chunks, rows in flight) instance that covers `cover` columns
#define LN_ROWS_PICK(T, CALL)                                             \
  do {                                                                    \
    constexpr int vec__ = rv::traits<T>::VEC;                             \
    const int tpr__ = ln::rows_threads(cover, vec__);                     \
    const int k__ = (cover + tpr__ * vec__ - 1) / (tpr__ * vec__);        \
    if (tpr__ == 1) CALL(T, 1, 1, 2);                                     \
    else if (tpr__ == 2) CALL(T, 2, 1, 2);                                \
    else if (tpr__ == 4) CALL(T, 4, 1, 2);                                \
    else if (tpr__ == 8) CALL(T, 8, 1, 2);                                \
    else if (tpr__ == 16) CALL(T, 16, 1, 2);                              \
    else if (tpr__ == 32) CALL(T, 32, 1, 2);                              \
    else if (tpr__ == 64 && k__ == 1) CALL(T, 64, 1, 2);                  \
    else if (tpr__ == 64 && k__ == 2) CALL(T, 64, 2, 1);                  \
    else if (tpr__ == 64) CALL(T, 64, 4, 1);                              \
    else if (vec__ == 8 || k__ <= 4) CALL(T, 256, 4, 1);                  \
    else CALL(T, 256, (vec__ == 8 ? 4 : 8), 1);                           \
  } while (0)

// part [parts][2 C] -> dweight, dbias (layer_norm_grad.hip)
int sum_parts(int parts, int C, const float* part, float* dw, float* db, hipStream_t st);

}  // namespace ln
