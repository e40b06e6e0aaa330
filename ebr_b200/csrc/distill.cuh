// distill.cuh: the distillation loss on a teacher's top logits and its gradient (formulas: include/ebr_tokens.h).
//
// A group of threads serves one row: the row's largest logit and sum of exponentials in one pass (running maximum and
// sum per thread, joined over the group), the loss from the K entries, and the gradient in a second pass over the row.
// The gradient of the entries' logits is written by the thread that owns the entry after the dense pass: it adds up the
// p of all entries with its id, in their order, so entries that repeat an id all write the same value.
//
// Exponentials are 2^((s - largest) * log2(e) / tau): the difference is taken before the scaling, so the exponent of a
// term that counts is exact to a few ulp, and the largest term is exactly 1.
#pragma once

#include "../../include/ebr_tokens.h"
#include "embedding.cuh"

namespace ebr {
namespace distill {

using embed::load_f;
using embed::store_f;

struct Args {
  int64_t N, V;
  int K;
  float tau, inv_tau, exp2_scale;  // exp2_scale = log2(e) / tau
  float factor;
  const void* logits;
  int64_t logits_stride;
  const void* top_ids;
  int ids64;
  const void* top_logits;
  int top_dtype;
  const float* row_weight;
  const float* upstream;  // gradient alone: NULL or one factor (stride 0) or one per row (stride 1)
  int64_t upstream_stride;
  int unless_one;
  float* losses;
  float* stats;
  void* grad;
};

__device__ __forceinline__ float top_value(const Args& a, int64_t i) {
  switch (a.top_dtype) {
    case EBR_FLOAT16: return __half2float(static_cast<const __half*>(a.top_logits)[i]);
    case EBR_BFLOAT16: return __bfloat162float(static_cast<const __nv_bfloat16*>(a.top_logits)[i]);
    default: return static_cast<const float*>(a.top_logits)[i];
  }
}

__device__ __forceinline__ int top_id(const Args& a, int64_t i) {  // -1: no entry
  if (a.ids64) {
    const int64_t v = static_cast<const int64_t*>(a.top_ids)[i];
    return v >= 0 && v < a.V ? static_cast<int>(v) : -1;
  }
  const int v = static_cast<const int*>(a.top_ids)[i];
  return v >= 0 && v < a.V ? v : -1;
}

// Sums and maxima over a group of kThreads threads (a warp or a block); every thread gets the result.
template <int kThreads>
struct Group {
  static constexpr int kWarps = kThreads / 32;
  float* red;  // kWarps floats (blocks)
  __device__ __forceinline__ void sync() const {
    if constexpr (kWarps == 1) __syncwarp(); else __syncthreads();
  }
  __device__ __forceinline__ float sum(float v) const {
    v = layers::warp_sum(v);
    if constexpr (kWarps > 1) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = red[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) v += red[w];
    }
    return v;
  }
  // NaN wins, as in the row maximum of a softmax over a row with a NaN.
  __device__ __forceinline__ static float larger(float a, float b) { return a > b || isnan(a) ? a : b; }
  __device__ __forceinline__ float max(float v) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = larger(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (kWarps > 1) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = red[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) v = larger(v, red[w]);
    }
    return v;
  }
};

// The teacher's probabilities of one row in shared memory: id[k] (-1: none) and p[k]. Returns whether there is an entry
// with p > 0 and, in entropy, sum p log p.
template <int kThreads>
__device__ __forceinline__ bool teacher_row(const Args& a, int64_t n, const Group<kThreads>& grp, int lane, int* id,
                                            float* p, float* entropy) {
  float top = -INFINITY;
  for (int k = lane; k < a.K; k += kThreads) {
    const int i = top_id(a, n * a.K + k);
    const float t = i >= 0 ? top_value(a, n * a.K + k) : -INFINITY;
    id[k] = i;
    p[k] = t;
    top = Group<kThreads>::larger(top, t);
  }
  top = grp.max(top);
  *entropy = 0.f;
  if (top == -INFINITY) return false;
  float total = 0.f;
  for (int k = lane; k < a.K; k += kThreads) total += exp2f((p[k] - top) * a.exp2_scale);
  total = grp.sum(total);
  const float log_total = logf(total), inv_total = 1.f / total;
  float e = 0.f;
  for (int k = lane; k < a.K; k += kThreads) {
    const float d = p[k] - top, q = exp2f(d * a.exp2_scale) * inv_total;
    if (q > 0.f || isnan(q)) e += q * (d * a.inv_tau - log_total);
    p[k] = q;
  }
  *entropy = grp.sum(e);
  grp.sync();
  return true;
}

// kStats: find the row's statistics and loss (else read the statistics). The group is the block (kThreads > 32) or one
// warp of a block of several. V vectors need rows that start on vector boundaries.
template <typename T, int kThreads, int kVec, bool kStats>
__global__ void distill_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[32];
  constexpr int kGroups = kThreads == 32 ? 8 : 1;
  const int group = kThreads == 32 ? threadIdx.x >> 5 : 0;
  const int lane = kThreads == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  if (n >= a.N) return;
  int* id = reinterpret_cast<int*>(smem) + group * 2 * a.K;
  float* p = reinterpret_cast<float*>(id + a.K);
  const Group<kThreads> grp{red};
  float up = 1.f;
  if (a.upstream) {
    up = a.upstream[n * a.upstream_stride];
    if (a.unless_one && up == 1.f) return;
  }
  const float weight = a.row_weight ? a.row_weight[n] : 1.f;
  float entropy;
  const bool any = teacher_row<kThreads>(a, n, grp, lane, id, p, &entropy) && weight != 0.f;
  const T* row = static_cast<const T*>(a.logits) + n * a.logits_stride;
  T* grad = a.grad ? static_cast<T*>(a.grad) + n * a.V : nullptr;
  if (!any) {
    if (kStats && lane == 0) {
      a.losses[n] = 0.f;
      if (a.stats) {
        a.stats[2 * n] = 0.f;
        a.stats[2 * n + 1] = 1.f;
      }
    }
    if (grad) {
      float z[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) z[i] = 0.f;
      for (int64_t c = static_cast<int64_t>(lane) * kVec; c < a.V; c += kThreads * kVec) store_f<T, kVec>(grad + c, z);
    }
    return;
  }
  float top, sum;
  if constexpr (kStats) {
    float m = -INFINITY, s = 0.f;
    for (int64_t c = static_cast<int64_t>(lane) * kVec; c < a.V; c += kThreads * kVec) {
      float v[kVec];
      load_f<T, kVec>(row + c, v);
      float vm = v[0];
#pragma unroll
      for (int i = 1; i < kVec; ++i) vm = Group<kThreads>::larger(vm, v[i]);
      if (vm > m || isnan(vm)) {
        s = m == -INFINITY ? 0.f : s * exp2f((m - vm) * a.exp2_scale);
        m = vm;
      }
      if (m != -INFINITY) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) s += exp2f((v[i] - m) * a.exp2_scale);
      }
    }
    top = grp.max(m);
    sum = grp.sum(m == -INFINITY ? 0.f : s * exp2f((m - top) * a.exp2_scale));
    if (top == -INFINITY) sum = NAN;  // a softmax over nothing
    const float log_sum = logf(sum);
    float cross = 0.f;
    for (int k = lane; k < a.K; k += kThreads) {
      if (id[k] < 0 || p[k] == 0.f) continue;
      cross += p[k] * ((Elem<T>::load(row + id[k]) - top) * a.inv_tau - log_sum);
    }
    cross = grp.sum(cross);
    if (lane == 0) {
      a.losses[n] = weight * (a.tau * a.tau) * (entropy - cross);
      if (a.stats) {
        a.stats[2 * n] = top;
        a.stats[2 * n + 1] = sum;
      }
    }
  } else {
    top = a.stats[2 * n];
    sum = a.stats[2 * n + 1];
  }
  if (!grad) return;
  const float coef = a.factor * up * weight * a.tau, inv_sum = 1.f / sum;
  for (int64_t c = static_cast<int64_t>(lane) * kVec; c < a.V; c += kThreads * kVec) {
    float v[kVec];
    load_f<T, kVec>(row + c, v);
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = coef * (exp2f((v[i] - top) * a.exp2_scale) * inv_sum);
    store_f<T, kVec>(grad + c, v);
  }
  grp.sync();
  for (int k = lane; k < a.K; k += kThreads) {
    if (id[k] < 0) continue;
    float mass = 0.f;
    for (int j = 0; j < a.K; ++j)
      if (id[j] == id[k]) mass += p[j];
    const float q = exp2f((Elem<T>::load(row + id[k]) - top) * a.exp2_scale) * inv_sum;
    grad[id[k]] = Elem<T>::to(coef * (q - mass));
  }
}

// total = factor * sum of the rows' losses, one block, a fixed order.
__global__ void __launch_bounds__(1024) total_kernel(int64_t N, float factor, const float* __restrict__ losses,
                                                     float* __restrict__ total) {
  __shared__ float red[32];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < N; i += 1024) s += losses[i];
  s = Group<1024>{red}.sum(s);
  if (threadIdx.x == 0) *total = factor * s;
}

}  // namespace distill
}  // namespace ebr
