// experts.cuh: tokens to their experts' rows and back, for a route made by key_sort.cuh.
//
//   scatter:  rows_out[row_of[t, k]] = w[t, k] * x[t]      (dispatch, and the gradient of combine's rows)
//             dots[t, k] = <x[t], rows_in[row_of[t, k]]>   (the gradient of combine's weights)
//   combine:  y[t] = sum_k w[t, k] * rows_in[row_of[t, k]] (combine, and the gradient of dispatch)
//
// All are bound by HBM. A warp serves one token, so that x[t] is read once for its K rows and y[t] is written once, and
// every access is a whole 16-byte vector per lane of one row. Rows of no slot are zeroed by further blocks of the same
// launch.
#pragma once

#include "embedding.cuh"

namespace ebr {
namespace experts {

using embed::load_f;
using embed::store_f;

constexpr int kWarps = 8;
constexpr int kZeroRows = 64;  // rows that a zeroing block looks at

template <typename T, typename TW, int V, bool kDots>
__global__ void __launch_bounds__(kWarps * 32) scatter_kernel(int64_t T_, int K, int64_t C, int64_t rows,
                                                              const T* __restrict__ x, int64_t x_stride,
                                                              const int* __restrict__ row_of,
                                                              const int* __restrict__ slot_of,
                                                              const TW* __restrict__ weights,
                                                              const T* __restrict__ rows_in, T* __restrict__ rows_out,
                                                              TW* __restrict__ dots, int token_blocks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) >= token_blocks) {
    const int64_t r0 = static_cast<int64_t>(blockIdx.x - token_blocks) * kZeroRows;
    for (int64_t r = r0 + warp; r < min(rows, r0 + kZeroRows); r += kWarps) {
      if (slot_of[r] >= 0) continue;
      float z[V];
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = 0.f;
      for (int64_t c = lane * V; c < C; c += 32 * V) store_f<T, V>(rows_out + r * C + c, z);
    }
    return;
  }
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (t >= T_) return;
  const T* xt = x + t * x_stride;
  if constexpr (kDots) {
    for (int k = 0; k < K; ++k) {
      const int row = row_of[t * K + k];
      float dot = 0.f;
      if (row >= 0) {
        const float w = weights ? Elem<TW>::load(weights + t * K + k) : 1.f;
        for (int64_t c = lane * V; c < C; c += 32 * V) {
          float a[V], b[V];
          load_f<T, V>(xt + c, a);
          load_f<T, V>(rows_in + static_cast<int64_t>(row) * C + c, b);
#pragma unroll
          for (int i = 0; i < V; ++i) dot += a[i] * b[i];
          if (rows_out) {
#pragma unroll
            for (int i = 0; i < V; ++i) a[i] *= w;
            store_f<T, V>(rows_out + static_cast<int64_t>(row) * C + c, a);
          }
        }
        dot = layers::warp_sum(dot);
      }
      if (lane == 0) dots[t * K + k] = Elem<TW>::to(dot);
    }
  } else {
    for (int64_t c = lane * V; c < C; c += 32 * V) {
      float a[V];
      load_f<T, V>(xt + c, a);
      for (int k = 0; k < K; ++k) {
        const int row = row_of[t * K + k];
        if (row < 0) continue;
        float b[V];
        const float w = weights ? Elem<TW>::load(weights + t * K + k) : 1.f;
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] = a[i] * w;
        store_f<T, V>(rows_out + static_cast<int64_t>(row) * C + c, b);
      }
    }
  }
}

template <typename T, typename TW, int V>
__global__ void __launch_bounds__(kWarps * 32) combine_kernel(int64_t T_, int K, int64_t C,
                                                              const T* __restrict__ rows_in, int64_t rows_stride,
                                                              const int* __restrict__ row_of,
                                                              const TW* __restrict__ weights, T* __restrict__ y) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (t >= T_) return;
  for (int64_t c = lane * V; c < C; c += 32 * V) {
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int k = 0; k < K; ++k) {
      const int row = row_of[t * K + k];
      if (row < 0) continue;
      const float w = weights ? Elem<TW>::load(weights + t * K + k) : 1.f;
      float b[V];
      load_f<T, V>(rows_in + row * rows_stride + c, b);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += w * b[i];
    }
    store_f<T, V>(y + t * C + c, acc);
  }
}

}  // namespace experts
}  // namespace ebr
