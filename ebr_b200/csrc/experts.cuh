// experts.cuh: tokens to their experts' rows and back, for a route made by key_sort.cuh.
//
//   scatter:  rows_out[row_of[t, k]] = w[t, k] * x[t]      (dispatch, and the gradient of combine's rows)
//             dots[t, k] = <x[t], rows_in[row_of[t, k]]>   (the gradient of combine's weights)
//   combine:  y[t] = sum_k w[t, k] * rows_in[row_of[t, k]] (combine, and the gradient of dispatch)
//
// All are bound by HBM. A warp serves one token, so that x[t] is read once for its K rows and y[t] is written once,
// and every access is a whole vector per lane of one row. kU vectors of a row, and those of several rows in the
// combine, are in flight at once; where the tokens are few, several warps (blockIdx.y) share a token's columns. The
// rows' numbers and weights of up to 32 slots sit in the lanes. Rows of no slot are zeroed by further blocks of the
// same launch.
//
// Measured, bfloat16: 16,384 tokens of 2,048 columns to eight of 64 experts: dispatch 107 us (5.7 TB/s), combine 96
// (6.3), combine's gradients 189 (6.1); the board batch (62,208 of 512, two of eight): 39, 39 and 62 us (4.8 to 5.1
// TB/s, a row of one kilobyte being two accesses of a warp). Rows of an odd number of 16-bit elements go two bytes a
// lane: 30,000 tokens of 1,001 to four of 32 take 74, 105 and 144 us (2.8 to 4.1 TB/s); reading them as shifted
// 16-byte windows was slower.
#pragma once

#include "embedding.cuh"

namespace ebr {
namespace experts {

using embed::Raw;
using embed::store_f;

constexpr int kWarps = 4;
constexpr int kZeroRows = 64;  // rows that a zeroing block looks at

// The slots k0 ... of token t: row numbers (-1 past the end) and weights, one per lane.
template <typename TW>
__device__ __forceinline__ void slots_of(const int* row_of, const TW* weights, int64_t t, int K, int k0, int lane,
                                         int* row, float* w) {
  const bool live = k0 + lane < K;
  *row = live ? row_of[t * K + k0 + lane] : -1;
  *w = live && weights && *row >= 0 ? Elem<TW>::load(weights + t * K + k0 + lane) : 1.f;
}

template <typename T, typename TW, int V, int kU, bool kDots>
__global__ void __launch_bounds__(kWarps * 32) scatter_kernel(int64_t T_, int K, int64_t C, int64_t rows,
                                                              const T* __restrict__ x, int64_t x_stride,
                                                              const int* __restrict__ row_of,
                                                              const int* __restrict__ slot_of,
                                                              const TW* __restrict__ weights,
                                                              const T* __restrict__ rows_in, T* __restrict__ rows_out,
                                                              TW* __restrict__ dots, int token_blocks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) >= token_blocks) {
    if (blockIdx.y > 0) return;
    const int64_t r0 = static_cast<int64_t>(blockIdx.x - token_blocks) * kZeroRows;
    for (int64_t r = r0 + warp; r < min(rows, r0 + kZeroRows); r += kWarps) {
      if (slot_of[r] >= 0) continue;
      const Raw<T, V> zero;
      for (int64_t c = lane * V; c < C; c += 32 * V) zero.store(rows_out + r * C + c);
    }
    return;
  }
  const int64_t step = static_cast<int64_t>(token_blocks) * kWarps;
  constexpr int64_t kTrip = int64_t{kU} * 32 * V;
  const int64_t first = blockIdx.y * kTrip, stride = gridDim.y * kTrip;
  int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  int my_row = -1, next_row;
  float my_w = 1.f, next_w;
  if (t < T_) slots_of(row_of, weights, t, K, 0, lane, &my_row, &my_w);
  for (; t < T_; t += step, my_row = next_row, my_w = next_w) {
    if (t + step < T_) slots_of(row_of, weights, t + step, K, 0, lane, &next_row, &next_w);
    const T* xt = x + t * x_stride;
    for (int k0 = 0; k0 < K; k0 += 32) {
      float my_dot = 0.f;
      if (k0 > 0) slots_of(row_of, weights, t, K, k0, lane, &my_row, &my_w);
      const int slots = min(32, K - k0);
      for (int64_t c0 = first + lane * V; c0 < C + lane * V; c0 += stride) {  // the same trips for all lanes
        Raw<T, V> a[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int64_t c = c0 + u * 32 * V;
          if (c < C) a[u].load(xt + c);
        }
        for (int k = 0; k < slots; ++k) {
          const int64_t row = __shfl_sync(0xffffffffu, my_row, k);
          const float w = __shfl_sync(0xffffffffu, my_w, k);
          if (row < 0) continue;
          Raw<T, V> b[kU];
          if constexpr (kDots) {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
              const int64_t c = c0 + u * 32 * V;
              if (c < C) b[u].load(rows_in + row * C + c);
            }
          }
          if (!kDots || rows_out) {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
              const int64_t c = c0 + u * 32 * V;
              if (c >= C) continue;
              if (weights) {
                float v[V];
                a[u].widen(v);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] *= w;
                store_f<T, V>(rows_out + row * C + c, v);
              } else {
                a[u].store(rows_out + row * C + c);
              }
            }
          }
          if constexpr (kDots) {
            float dot = 0.f;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
              float p[V], q[V];
              a[u].widen(p);
              b[u].widen(q);
#pragma unroll
              for (int i = 0; i < V; ++i) dot += p[i] * q[i];
            }
            dot = layers::warp_sum(dot);
            if (lane == k) my_dot += dot;
          }
        }
      }
      if (kDots && lane < slots) dots[t * K + k0 + lane] = Elem<TW>::to(my_dot);
    }
  }
}

template <typename T, typename TW, int V, int kU>
__global__ void __launch_bounds__(kWarps * 32) combine_kernel(int64_t T_, int K, int64_t C,
                                                              const T* __restrict__ rows_in, int64_t rows_stride,
                                                              const int* __restrict__ row_of,
                                                              const TW* __restrict__ weights, T* __restrict__ y) {
  constexpr int kRows = 2;  // rows in flight
  const int lane = threadIdx.x & 31;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  constexpr int64_t kTrip = int64_t{kU} * 32 * V;
  const int64_t first = blockIdx.y * kTrip, stride = gridDim.y * kTrip;
  int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  int my_row = -1, next_row;
  float my_w = 1.f, next_w;
  if (t < T_) slots_of(row_of, weights, t, K, 0, lane, &my_row, &my_w);
  for (; t < T_; t += step, my_row = next_row, my_w = next_w) {
    if (t + step < T_) slots_of(row_of, weights, t + step, K, 0, lane, &next_row, &next_w);
    for (int64_t c0 = first + lane * V; c0 < C + lane * V; c0 += stride) {  // the same trips for all lanes
      float acc[kU][V];
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[u][i] = 0.f;
      for (int k0 = 0; k0 < K; k0 += 32) {
        if (K > 32) slots_of(row_of, weights, t, K, k0, lane, &my_row, &my_w);
        const int slots = min(32, K - k0);
        for (int k = 0; k < slots; k += kRows) {
          Raw<T, V> b[kRows][kU];
          float w[kRows];
          int row[kRows];
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            row[r] = __shfl_sync(0xffffffffu, my_row, (k + r) & 31);
            w[r] = __shfl_sync(0xffffffffu, my_w, (k + r) & 31);
            if (k + r >= slots) row[r] = -1;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
              // Lanes past the row and dropped slots read somewhere valid: no branch stands between the loads.
              const int64_t c = c0 + u * 32 * V;
              b[r][u].load(rows_in + max(row[r], 0) * rows_stride + (c < C ? c : 0));
            }
          }
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            if (row[r] < 0) continue;  // a dropped slot adds nothing, not 0 * its weight
#pragma unroll
            for (int u = 0; u < kU; ++u) {
              float v[V];
              b[r][u].widen(v);
#pragma unroll
              for (int i = 0; i < V; ++i) acc[u][i] += w[r] * v[i];
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int64_t c = c0 + u * 32 * V;
        if (c < C) store_f<T, V>(y + t * C + c, acc[u]);
      }
    }
  }
}

}  // namespace experts
}  // namespace ebr
