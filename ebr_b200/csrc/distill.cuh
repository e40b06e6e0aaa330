// distill.cuh: the distillation loss on a teacher's top logits and its gradient (formulas: include/ebr_tokens.h).
//
// A row of a few logits takes four lanes, one of up to 32 KB a warp, a longer one a CTA or a cluster with the row in
// a shared-memory ring. The gradient of the logits that the teacher names is written after the dense pass.
//
// Exponentials are 2^((s - largest) * log2(e) / tau): the difference is taken before the scaling, so the exponent of
// a term that counts is exact to a few ulp, and the largest term is exactly 1. Logarithms are taken times tau, and the
// loss is tau times their sum: neither 1 / tau nor tau^2 is formed, which leave float32 at temperatures (and at masked
// logits) whose losses do not.
//
// Measured, bfloat16, 64 entries, loss and gradient in one pass: 4,096 rows of 131,072 take 436 to 444 us (4.8 TB/s of
// logits and gradient; the loss alone 202, 5.3 TB/s; the gradient alone 348, 6.2 TB/s), 16,384 of 32,768 504 us,
// 65,536 of 8,192 515 us, 131,072 of 4,096 (16 entries) 394 us (5.5 TB/s). The one-pass kernel is bound by latency,
// issue and the exponential unit together (61 and 58 % busy with the 24 warps that the rings leave room for on an SM).
// The warp kernel misses L2 at its second reading of rows of 8 to 32 KB: at 8,192 rows of 16,384 it reads 594 MB from
// HBM for 268 MB of logits. Rows whose gradient starts at another place of a 16-byte word (a view of rows that are more
// than 256 elements longer, by a number that is no multiple of 16 bytes) are stored element by element: 8,388 rows of
// 32,001 take 868 us so, 269 where the places agree.
#pragma once

#include "../../include/ebr_tokens.h"
#include "embedding.cuh"

namespace ebr {
namespace distill {

struct Args {
  int64_t N, V;
  int K;
  float tau, exp2_scale;  // exp2_scale = log2(e) / tau
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
  int64_t grad_stride;
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

// 2^((v + base) * scale) of a pair, the sum and the product as packed instructions: the one-pass kernel is short of
// issue slots (an earlier form of it took 505 us with them on rows of 131,072, 520 without).
__device__ __forceinline__ float2 exp2_pair(float2 v, float base, float scale) {
  float2 d;
  asm("{.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmul.rn.f32x2 x, x, z;\n\tmov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(v.x), "f"(v.y), "f"(base), "f"(scale));
  return make_float2(exp2_approx(d.x), exp2_approx(d.y));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }

// A 16-byte granule of logits as pairs of floats, the larger elements of two granules place by place and the largest
// of one (NaN passed over), and pairs back to a granule.
template <typename T>
struct Granule;
template <>
struct Granule<float> {
  static constexpr int kPairs = 2;
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }  // -inf
  static __device__ __forceinline__ void split(const uint4& g, float2 (&v)[2]) {
    v[0] = make_float2(__uint_as_float(g.x), __uint_as_float(g.y));
    v[1] = make_float2(__uint_as_float(g.z), __uint_as_float(g.w));
  }
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
    uint4 r;
    r.x = __float_as_uint(fmaxf(__uint_as_float(a.x), __uint_as_float(b.x)));
    r.y = __float_as_uint(fmaxf(__uint_as_float(a.y), __uint_as_float(b.y)));
    r.z = __float_as_uint(fmaxf(__uint_as_float(a.z), __uint_as_float(b.z)));
    r.w = __float_as_uint(fmaxf(__uint_as_float(a.w), __uint_as_float(b.w)));
    return r;
  }
  static __device__ __forceinline__ float largest(const uint4& g) {
    return fmaxf(fmaxf(__uint_as_float(g.x), __uint_as_float(g.y)), fmaxf(__uint_as_float(g.z), __uint_as_float(g.w)));
  }
  static __device__ __forceinline__ uint4 join(const float2 (&v)[2]) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
};
template <>
struct Granule<__nv_bfloat16> {
  static constexpr int kPairs = 4;
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }  // -inf
  static __device__ __forceinline__ float2 pair(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void split(const uint4& g, float2 (&v)[4]) {
    v[0] = pair(g.x);
    v[1] = pair(g.y);
    v[2] = pair(g.z);
    v[3] = pair(g.w);
  }
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
    const __nv_bfloat162 *x = reinterpret_cast<const __nv_bfloat162*>(&a), *y = reinterpret_cast<const __nv_bfloat162*>(&b);
    uint4 r;
    __nv_bfloat162* z = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = __hmax2(x[i], y[i]);
    return r;
  }
  static __device__ __forceinline__ float largest(const uint4& g) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&g);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const float2 f = pair(*reinterpret_cast<const uint32_t*>(&m));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ uint4 join(const float2 (&v)[4]) {
    uint4 g;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&g);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __float22bfloat162_rn(v[i]);
    return g;
  }
};
template <>
struct Granule<__half> {
  static constexpr int kPairs = 4;
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }  // -inf
  static __device__ __forceinline__ void split(const uint4& g, float2 (&v)[4]) {
    const __half2* h = reinterpret_cast<const __half2*>(&g);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __half22float2(h[i]);
  }
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
    const __half2 *x = reinterpret_cast<const __half2*>(&a), *y = reinterpret_cast<const __half2*>(&b);
    uint4 r;
    __half2* z = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = __hmax2(x[i], y[i]);
    return r;
  }
  static __device__ __forceinline__ float largest(const uint4& g) {
    const __half2* h = reinterpret_cast<const __half2*>(&g);
    const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ uint4 join(const float2 (&v)[4]) {
    uint4 g;
    __half2* h = reinterpret_cast<__half2*>(&g);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __float22half2_rn(v[i]);
    return g;
  }
};

// The sum of 2^((v + base) * scale) over a granule.
template <typename T>
__device__ __forceinline__ float exp2_sum(const uint4& g, float base, float scale) {
  float2 v[Granule<T>::kPairs];
  Granule<T>::split(g, v);
#pragma unroll
  for (int i = 0; i < Granule<T>::kPairs; ++i) v[i] = exp2_pair(v[i], base, scale);
#pragma unroll
  for (int w = Granule<T>::kPairs / 2; w > 0; w /= 2)
#pragma unroll
    for (int i = 0; i < w; ++i) v[i] = add2(v[i], v[i + w]);
  return v[0].x + v[0].y;
}

// A maximum and the sum of 2^((v - maximum) * scale). Maxima pass NaN over (an instruction less per element); a NaN
// makes the sum NaN, and with it the row's loss and gradient, all the same.
struct Stat {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : -m; }  // terms of -inf are 0, not NaN
  // The sum with another maximum `top` >= m.
  __device__ __forceinline__ float sum_at(float top, float scale) const {
    return m == -INFINITY ? s : s * exp2_approx((m - top) * scale);
  }
};

// A row that does not count (no entry of the teacher, or weight 0) has this sum among the statistics: no other row
// can.
__device__ __forceinline__ float2 no_row() { return make_float2(0.f, INFINITY); }

// Sum over the kLanes consecutive lanes of a group.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int kLanes>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// The largest over the warp, in every lane, by one instruction.
__device__ __forceinline__ float warp_largest(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// ------------------------------------------------------------------------------------------------ short rows

// kLanes lanes serve a row; a row is short enough for its second and third reading to come from L1. The teacher's
// entries are in shared memory, kSmallThreads / kLanes rows' worth.
constexpr int kSmallThreads = 256;

template <typename T, int kLanes, bool kStats>
__global__ void __launch_bounds__(kSmallThreads) distill_small_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int kGroups = kSmallThreads / kLanes;
  if (!kStats && a.unless_one && a.upstream[0] == 1.f) return;
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  const bool live = n < a.N;  // lanes of no row stay for the shuffles
  int* id = reinterpret_cast<int*>(smem) + group * 2 * a.K;
  float* p = reinterpret_cast<float*>(id + a.K);
  const float weight = !live ? 0.f : a.row_weight ? a.row_weight[n] : 1.f;
  const unsigned group_lanes = kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u) << (threadIdx.x % 32 / kLanes * kLanes);
  float top = -INFINITY;
  bool entry = false;
  for (int k = lane; k < a.K; k += kLanes) {
    const int i = live ? top_id(a, n * a.K + k) : -1;
    const float t = i >= 0 ? top_value(a, n * a.K + k) : -INFINITY;
    id[k] = i;
    p[k] = t;
    top = fmaxf(top, t);
    entry |= t != -INFINITY;
  }
  top = lanes_max<kLanes>(top);
  entry = __any_sync(group_lanes, entry);
  const bool any = entry && weight != 0.f;
  float total = 0.f;
  if (any)
    for (int k = lane; k < a.K; k += kLanes) total += exp2_approx((p[k] - top) * a.exp2_scale);
  total = lanes_sum<kLanes>(total);
  const float log_total = logf(total), inv_total = 1.f / total;
  const T* row = static_cast<const T*>(a.logits) + n * a.logits_stride;
  Stat st;
  if (kStats) {
    if (any)
      for (int64_t c = lane; c < a.V; c += kLanes) st.m = fmaxf(st.m, Elem<T>::load(row + c));
    st.m = lanes_max<kLanes>(st.m);
    const float base = st.base();
    if (any)
      for (int64_t c = lane; c < a.V; c += kLanes) st.s += exp2_approx((Elem<T>::load(row + c) + base) * a.exp2_scale);
    st.s = lanes_sum<kLanes>(st.s);
    if (st.m == -INFINITY) st.s = NAN;  // a softmax over nothing
  } else if (any) {
    st.m = a.stats[2 * n];
    st.s = a.stats[2 * n + 1];
  }
  float loss = 0.f;
  if (any) {
    const float log_sum = logf(st.s);
    for (int k = lane; k < a.K; k += kLanes) {
      // No entry, no probability: 0 times a total of NaN (a teacher's logit of NaN or infinity) is not 0.
      const float d = p[k] - top, q = id[k] >= 0 ? exp2_approx(d * a.exp2_scale) * inv_total : 0.f;
      p[k] = q;
      if (kStats && (q > 0.f || isnan(q)))
        loss += q * ((d - a.tau * log_total) - ((Elem<T>::load(row + id[k]) - st.m) - a.tau * log_sum));
    }
  }
  if (kStats) {
    loss = lanes_sum<kLanes>(loss);
    if (live && lane == 0) {
      a.losses[n] = any ? weight * a.tau * loss : 0.f;
      if (a.stats) {
        reinterpret_cast<float2*>(a.stats)[n] = any ? make_float2(st.m, st.s) : no_row();
      }
    }
  }
  __syncwarp();  // the group's probabilities are complete
  if (!live || !a.grad) return;
  T* grad = static_cast<T*>(a.grad) + n * a.grad_stride;
  const float up = a.upstream ? a.upstream[n * a.upstream_stride] : 1.f;
  const float coef = a.factor * up * weight * a.tau, inv_sum = 1.f / st.s;
  for (int64_t c = lane; c < a.V; c += kLanes) {
    float g = 0.f;
    if (any) {
      g = exp2_approx((Elem<T>::load(row + c) - st.m) * a.exp2_scale) * inv_sum;
      float mass = 0.f;
      for (int k = 0; k < a.K; ++k)
        if (id[k] == c) mass += p[k];
      g = coef * (g - mass);
    }
    grad[c] = Elem<T>::to(g);
  }
}

// ------------------------------------------------------------------------------------------------ long rows

// A row in 16-byte granules of memory: element j sits at place phase + j of the granules, so that whole granules are
// aligned whatever the row's start; the first and last may hold fewer elements of the row.
template <typename T>
struct Granules {
  static constexpr int kE = static_cast<int>(16 / sizeof(T));
  const T* row;
  int phase, V;  // V <= 2^19
  __device__ __forceinline__ Granules(const T* r, int64_t v) : row(r), V(static_cast<int>(v)) {
    phase = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
  }
  __device__ __forceinline__ int count() const { return (phase + V + kE - 1) / kE; }
  __device__ __forceinline__ bool whole(int g) const {
    return (g > 0 || phase == 0) && (g + 1) * kE <= phase + V;
  }
  // Whole granules [first_whole, end_whole), when there is one.
  __device__ __forceinline__ int first_whole() const { return phase ? 1 : 0; }
  __device__ __forceinline__ int end_whole() const { return (phase + V) / kE; }
  __device__ __forceinline__ int first(int g) const { return g * kE - phase; }  // element
  // The ragged granule at the front (end 0) or at the back (end 1), -1 where there is none or another `end`.
  __device__ __forceinline__ int ragged_end(int end) const {
    const int g = end == 0 ? 0 : end == 1 ? count() - 1 : -1;
    return g >= end && !whole(g) ? g : -1;
  }
};

// mult * 2^((v - m) * scale) for a granule.
template <typename T>
__device__ __forceinline__ uint4 grad_granule(const uint4& raw, float m, float scale, float mult) {
  float2 v[Granule<T>::kPairs];
  Granule<T>::split(raw, v);
#pragma unroll
  for (int i = 0; i < Granule<T>::kPairs; ++i) v[i] = mul2(exp2_pair(v[i], -m, scale), make_float2(mult, mult));
  return Granule<T>::join(v);
}

// The elements of a granule that belong to the row, one by one, from element j0 on.
template <typename T>
__device__ __forceinline__ void store_elements(const uint4& g, int j0, int V, T* row) {
  constexpr int kE = static_cast<int>(16 / sizeof(T));
  const layers::Pack<T, kE> e = *reinterpret_cast<const layers::Pack<T, kE>*>(&g);
#pragma unroll
  for (int i = 0; i < kE; ++i)
    if (j0 + i >= 0 && j0 + i < V) row[j0 + i] = e.e[i];
}

template <typename T>
__device__ __forceinline__ uint4 ragged(const Granules<T>& r, int g) {  // the row's elements of a granule, else -inf
  constexpr int kE = Granules<T>::kE;
  layers::Pack<T, kE> v;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const int j = r.first(g) + i;
    v.e[i] = j >= 0 && j < r.V ? r.row[j] : Elem<T>::to(-INFINITY);
  }
  return *reinterpret_cast<const uint4*>(&v);
}

// Untiled TMA copies: both addresses and the size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(smem_dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* smem_src, uint32_t bytes, uint64_t policy) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group.L2::cache_hint [%0], [%1], %2, %3;" ::"l"(dst),
               "r"(smem_u32(smem_src)), "r"(bytes), "l"(policy)
               : "memory");
}
// L2 policies: what will not be read again soon, and what will.
__device__ __forceinline__ uint64_t policy_once() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t policy_again() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// Wait until all but the newest kLeft committed stores of this thread have finished reading shared memory.
template <int kLeft>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kLeft) : "memory");
}

// What the waits of distill_row_kernel record when they run out; they go on then, so that nothing hangs.
constexpr int kFullWaitSite = 7001, kEmptyWaitSite = 7002, kExchangeWaitSite = 7003;

// The statistics of one warp, and their announcement on an mbarrier, in the shared memory of CTA `rank` of the
// cluster.
__device__ __forceinline__ void push_stat(float2* slot, uint64_t* bar, uint32_t rank, float m, float s) {
  asm volatile(
      "{\n\t.reg .b32 a, b;\n\t"
      "mapa.shared::cluster.u32 a, %0, %2;\n\t"
      "mapa.shared::cluster.u32 b, %1, %2;\n\t"
      "st.shared::cluster.v2.f32 [a], {%3, %4};\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [b];\n\t}" ::"r"(smem_u32(slot)),
      "r"(smem_u32(bar)), "r"(rank), "f"(m), "f"(s)
      : "memory");
}

// mbar_wait for what other CTAs of the cluster have written.
__device__ __forceinline__ void wait_cluster(uint64_t* bar, uint32_t parity, int site) {
  const uint32_t addr = smem_u32(bar);
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 1;; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return;
    if ((i & 255u) == 0 && globaltimer_ns() - t0 > kWaitLimitNs) {
      atomicExch(&g_device_error, site);
      return;
    }
  }
}

constexpr int kMaxSlices = 16;

// The two halves of a cluster barrier, for the one that only makes sure that every CTA of the cluster runs before its
// shared memory is written from another.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Zeros for the granules [lo, hi) of a gradient row, by the block's first `threads` threads.
template <typename T>
__device__ __forceinline__ void zero_granules(const Granules<T>& r, int lo, int hi, int threads, T* grad) {
  const layers::Pack<T, Granules<T>::kE> z = {};
  for (int g = lo + threadIdx.x; g < hi; g += threads) {
    const int j0 = r.first(g);
    if (r.whole(g)) {
      *reinterpret_cast<layers::Pack<T, Granules<T>::kE>*>(grad + j0) = z;
    } else {
      for (int i = 0; i < Granules<T>::kE; ++i)
        if (j0 + i >= 0 && j0 + i < r.V) grad[j0 + i] = z.e[i];
    }
  }
}

// Row n's weight, 0 where it has no entry: what the dense kernel has to know of the teacher. By a whole warp.
__device__ __forceinline__ float weight_by_warp(const Args& a, int64_t n) {
  bool any = false;
  for (int k = threadIdx.x & 31; k < a.K; k += 32) {
    const int i = top_id(a, n * a.K + k);
    const float t = top_value(a, n * a.K + k);
    any |= i >= 0 && t != -INFINITY;
  }
  return !__any_sync(0xffffffffu, any) ? 0.f : a.row_weight ? a.row_weight[n] : 1.f;
}

// The same for all rows, before the dense kernel, because there the dependent reads would stand in every row's way.
__global__ void __launch_bounds__(256) distill_weights_kernel(const __grid_constant__ Args a, float* weights) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (n >= a.N) return;
  const float w = weight_by_warp(a, n);
  if ((threadIdx.x & 31) == 0) weights[n] = w;
}

// The dense part of long rows: the statistics, and grad = c_n q where a.grad is set, so that the logits cross HBM
// once. CTA `slice` of a cluster of `slices` (one, unless the rows are few) serves a slice of the row's granules, in
// chunks of kU granules for each lane, which pass through a ring of `slots` chunks in shared memory. The last warp
// loads (TMA); the others reduce a row's chunks in order, exchange their statistics, and then turn the chunks into
// the gradient in place and store them (TMA), each warp its own part of a chunk, so that within a row the warps meet
// only for the exchange. The last chunks of a row stay in the ring between the two passes; only what does not fit is
// loaded again, soon after its first reading, from L2. While a row is in its second pass, the freed slots already
// take the next row. The chunks are freed in the order in which they were loaded, so the ring needs no bookkeeping
// but two counters. What needs the teacher's entries is left to distill_entries_kernel: here each warp of each CTA
// would pay for it.
constexpr int kMaxSlots = 16;

template <typename T, int kWarps, int kU>
__global__ void __launch_bounds__(kWarps * 32 + 32) distill_row_kernel(const __grid_constant__ Args a,
                                                                       const float* weights, int slices,
                                                                       int slice_granules, int slots) {
  constexpr int kParts = kMaxSlices * kWarps, kE = Granules<T>::kE;
  constexpr int kPart = kU * 32, kChunk = kPart * kWarps;  // granules of a warp's part of a chunk, of a chunk
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float2 stat[2][kParts];
  __shared__ uint64_t full[kMaxSlots], empty[kMaxSlots], exchanged[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = static_cast<int>(blockIdx.x) % slices;
  const int rows = static_cast<int>(a.N), step = static_cast<int>(gridDim.x) / slices;
  uint4* ring = reinterpret_cast<uint4*>(smem);
  // This CTA's whole granules of a row: `count` of them from element `begin` on. The row's ragged ends, at most two
  // of them in a slice, belong to lanes 0 and 1 of warp 0.
  struct Slice {
    const T* row;
    int begin, count, chunks, kept;
  };
  auto slice_of = [&](const Granules<T>& r) {
    const int lo = max(r.first_whole(), slice * slice_granules), hi = min(r.end_whole(), (slice + 1) * slice_granules);
    Slice s;
    s.row = r.row;
    s.begin = r.first(lo);
    s.count = max(0, hi - lo);
    s.chunks = (s.count + kChunk - 1) / kChunk;
    s.kept = a.grad ? min(s.chunks, slots - 2) : 0;
    return s;
  };
  auto row_of = [&](int n) { return Granules<T>(static_cast<const T*>(a.logits) + n * a.logits_stride, a.V); };

  if (threadIdx.x == 0) {
    for (int b = 0; b < slots; ++b) {
      mbar_init(&full[b], 1);
      mbar_init(&empty[b], kWarps);
    }
    mbar_init(&exchanged[0], slices * kWarps);
    mbar_init(&exchanged[1], slices * kWarps);
    fence_barrier_init();
  }
  __syncthreads();
  if (slices > 1) {
    cluster_arrive();
    cluster_wait();  // every CTA's barriers are there before another one arrives at them
  }
  const int first = static_cast<int>(blockIdx.x) / slices;
  // weights is NULL where no cluster has a second row: the warps then read the row's entries themselves
  const float own = weights ? 0.f : weight_by_warp(a, first);
  auto weight_of = [&](int n) { return weights ? weights[n] : own; };
  if (warp == kWarps) {
    if (lane == 0) {
      const uint64_t once = policy_once(), again = policy_again();
      int slot = 0, round = 0;
      for (int n = first; n < rows; n += step) {
        if (weight_of(n) == 0.f) continue;
        const Slice s = slice_of(row_of(n));
        const int loads = s.chunks + (a.grad ? s.chunks - s.kept : 0);
        for (int j = 0; j < loads; ++j) {
          const int c = j < s.chunks ? j : j - s.chunks;
          if (round > 0) mbar_wait(&empty[slot], (round - 1) & 1, kEmptyWaitSite);
          const uint32_t bytes = static_cast<uint32_t>(min(kChunk, s.count - c * kChunk)) * 16;
          mbar_arrive_expect_tx(&full[slot], bytes);
          bulk_load(ring + slot * kChunk, s.row + s.begin + c * kChunk * kE, bytes, &full[slot],
                    j < loads - s.chunks ? again : once);
          if (++slot == slots) slot = 0, ++round;
        }
      }
    }
  } else {
    const uint64_t once = policy_once();
    int slot = 0, round = 0, exchange = 0;
    auto advance = [&] {
      if (++slot == slots) slot = 0, ++round;
    };
    float weight = first < rows ? weight_of(first) : 0.f;
    for (int n = first; n < rows; n += step) {
      const float now = weight;
      weight = n + step < rows ? weight_of(n + step) : 0.f;
      T* grad = a.grad ? static_cast<T*>(a.grad) + n * a.grad_stride : nullptr;
      if (now == 0.f) {  // the same in every warp of the cluster
        if (grad) {
          const Granules<T> out(grad, a.V);
          const int span = (out.count() + slices - 1) / slices;
          zero_granules(out, min(out.count(), slice * span), min(out.count(), (slice + 1) * span), kWarps * 32, grad);
        }
        if (slice == 0 && threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[n] = no_row();
        continue;
      }
      const Granules<T> row = row_of(n);
      const Slice s = slice_of(row);
      int end = row.ragged_end(static_cast<int>(threadIdx.x));  // this thread's ragged granule
      if (end < slice * slice_granules || end >= (slice + 1) * slice_granules) end = -1;
      const uint4 ragged_end = end >= 0 ? ragged(row, end) : Granule<T>::none();
      // first pass: the statistics, the maximum the warp's own
      Stat st;
      const int part = warp * kPart + lane;
      int kept_slot = slot;
      for (int c = 0; c < s.chunks; ++c) {
        if (c == s.chunks - s.kept) kept_slot = slot;
        mbar_wait(&full[slot], round & 1, kFullWaitSite);
        const uint4* chunk = ring + slot * kChunk + part;
        const int left = s.count - c * kChunk - part;
        uint4 v[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) v[u] = chunk[u * 32];  // in the ring, if not of this row
        if (c + 1 == s.chunks)
#pragma unroll
          for (int u = 0; u < kU; ++u)
            if (u * 32 >= left) v[u] = Granule<T>::none();
        uint4 most = v[0];
#pragma unroll
        for (int u = 1; u < kU; ++u) most = Granule<T>::larger(most, v[u]);
        const float top = warp_largest(Granule<T>::largest(most));
        if (top > st.m) {
          st.s *= exp2_approx((st.m - top) * a.exp2_scale);
          st.m = top;
        }
        const float base = st.base();
#pragma unroll
        for (int u = 0; u < kU; ++u) st.s += exp2_sum<T>(v[u], base, a.exp2_scale);
        if (c < s.chunks - s.kept) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[slot]);
        }
        advance();
      }
      if (warp == 0) {
        const float top = warp_largest(Granule<T>::largest(ragged_end));
        if (top > st.m) {
          st.s *= exp2_approx((st.m - top) * a.exp2_scale);
          st.m = top;
        }
        st.s += exp2_sum<T>(ragged_end, st.base(), a.exp2_scale);
      }
      st.s = lanes_sum<32>(st.s);
      float2* mine = stat[exchange & 1];
      if (lane < slices) push_stat(mine + slice * kWarps + warp, &exchanged[exchange & 1], lane, st.m, st.s);
      wait_cluster(&exchanged[exchange & 1], exchange >> 1 & 1, kExchangeWaitSite);
      ++exchange;
      Stat all;
      float2 piece[kParts / 32];
#pragma unroll
      for (int u = 0; u < kParts / 32; ++u) {
        const int at = u * 32 + lane;
        piece[u] = at < slices * kWarps ? mine[at] : make_float2(-INFINITY, 0.f);
        all.m = fmaxf(all.m, piece[u].x);
        if ((u + 1) * 32 >= slices * kWarps) break;
      }
      all.m = warp_largest(all.m);
#pragma unroll
      for (int u = 0; u < kParts / 32; ++u) {
        const Stat one{piece[u].x, piece[u].y};
        all.s += one.sum_at(all.m, a.exp2_scale);
        if ((u + 1) * 32 >= slices * kWarps) break;
      }
      all.s = lanes_sum<32>(all.s);
      if (all.m == -INFINITY) all.s = NAN;  // a softmax over nothing
      if (slice == 0 && threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[n] = make_float2(all.m, all.s);
      if (!grad) continue;
      // second pass: the chunks that stayed, then the others again
      const float mult = a.factor * now * a.tau / all.s;
      const bool same = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
      int last = -1;  // lane 0: the slot whose store may still be read
      for (int j = 0; j < s.chunks; ++j) {
        const bool again = j >= s.kept;
        const int c = again ? j - s.kept : s.chunks - s.kept + j;
        const int at = again ? slot : kept_slot;
        if (again) {
          mbar_wait(&full[slot], round & 1, kFullWaitSite);
          advance();
        } else if (++kept_slot == slots) {
          kept_slot = 0;
        }
        uint4* chunk = ring + at * kChunk + part;
        const int left = s.count - c * kChunk - part, from = s.begin + (c * kChunk + part) * kE;
        uint4 v[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) v[u] = chunk[u * 32];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          v[u] = grad_granule<T>(v[u], all.m, a.exp2_scale, mult);
          if (u * 32 >= left) continue;
          if (same)
            chunk[u * 32] = v[u];
          else  // rows that start at different places of a 16-byte word
            store_elements<T>(v[u], from + u * 32 * kE, row.V, grad);
        }
        if (same) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          const int granules = min(kPart, s.count - c * kChunk - warp * kPart);
          if (same && granules > 0)
            bulk_store(grad + from, chunk, static_cast<uint32_t>(granules) * 16, once);
          tma_store_commit();
          if (last >= 0) {
            bulk_wait_read<1>();
            mbar_arrive(&empty[last]);
          }
          last = at;
        }
      }
      if (lane == 0 && last >= 0) {
        bulk_wait_read<0>();
        mbar_arrive(&empty[last]);
      }
      if (end >= 0)
        store_elements<T>(grad_granule<T>(ragged_end, all.m, a.exp2_scale, mult), row.first(end), row.V, grad);
    }
    if (lane == 0) tma_store_wait_all();
  }
  if (slices > 1) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();  // nobody leaves while its shared memory may be written
  }
}

// --------------------------------------------------------------------------------------------- the teacher's entries

// One row's entries, by one warp, in its shared memory: ids, logits that become probabilities, and a table of bits.
struct Entries {
  int* id;
  float* p;
  unsigned* seen;
  int lane;
  float top, log_total, inv_total;

  __device__ __forceinline__ Entries(void* smem, int K, int lane_) : lane(lane_) {
    id = static_cast<int*>(smem);
    p = reinterpret_cast<float*>(id + K);
    seen = reinterpret_cast<unsigned*>(p + K);
  }
  // Reads them; whether there is one.
  __device__ __forceinline__ bool read(const Args& a, int64_t n) {
    bool any = false;
    top = -INFINITY;
    for (int k = lane; k < a.K; k += 32) {
      const int i = top_id(a, n * a.K + k);
      const float v = top_value(a, n * a.K + k), t = i >= 0 ? v : -INFINITY;
      id[k] = i;
      p[k] = t;
      seen[k] = 0;
      any |= t != -INFINITY;
      top = fmaxf(top, t);
    }
    top = warp_largest(top);
    return __any_sync(0xffffffffu, any);
  }
  // p becomes the probabilities.
  __device__ __forceinline__ void normalise(const Args& a) {
    float total = 0.f;
    for (int k = lane; k < a.K; k += 32) total += exp2_approx((p[k] - top) * a.exp2_scale);
    total = lanes_sum<32>(total);
    log_total = logf(total);
    inv_total = 1.f / total;
  }
  // The row's loss over tau, from the statistics (m, log of the sum), in every lane; p must still be the logits.
  template <typename T, bool kLoss>
  __device__ __forceinline__ float finish(const Args& a, const T* row, float m, float log_sum) {
    float loss = 0.f;
    for (int k = lane; k < a.K; k += 32) {
      // No entry, no probability: 0 times a total of NaN (a teacher's logit of NaN or infinity) is not 0.
      const float d = p[k] - top, q = id[k] >= 0 ? exp2_approx(d * a.exp2_scale) * inv_total : 0.f;
      p[k] = q;
      if (kLoss && (q > 0.f || isnan(q)))
        loss += q * ((d - a.tau * log_total) - ((Elem<T>::load(row + id[k]) - m) - a.tau * log_sum));
    }
    return kLoss ? lanes_sum<32>(loss) : 0.f;
  }
  // The gradient of the logits that they name, over what the dense pass wrote. Entries that repeat an id share the
  // sum of their p: the table finds the entries that may be such (two ids can have one bit), and the warp adds up
  // each of those ids' p in the entries' order, so that the rest (nearly all) cost nothing.
  template <typename T>
  __device__ __forceinline__ void store(const Args& a, const T* row, float m, float inv_sum, float coef, T* grad) {
    const unsigned bits = 32u * static_cast<unsigned>(a.K);
    __syncwarp();
    for (int k0 = 0; k0 < a.K; k0 += 32) {
      const int mine = k0 + lane < a.K ? id[k0 + lane] : -1;
      bool again = false;
      if (mine >= 0) {
        const unsigned bit = static_cast<unsigned>(mine) * 2654435761u % bits;
        again = atomicOr(&seen[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1;
        const float q = exp2_approx((Elem<T>::load(row + mine) - m) * a.exp2_scale) * inv_sum;
        grad[mine] = Elem<T>::to(coef * (q - p[k0 + lane]));
      }
      for (unsigned todo = __ballot_sync(0xffffffffu, again); todo; todo &= todo - 1) {
        const int named = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
        float mass = 0.f;
        for (int j = lane; j < a.K; j += 32)
          if (id[j] == named) mass += p[j];
        mass = lanes_sum<32>(mass);
        __syncwarp();
        if (lane == 0) {
          const float q = exp2_approx((Elem<T>::load(row + named) - m) * a.exp2_scale) * inv_sum;
          grad[named] = Elem<T>::to(coef * (q - mass));
        }
      }
    }
  }
};

// The gradient alone, from the forward's statistics: its dense part, blocks walking over (row, slice) items; with
// kEntries (whole rows: one slice) the entries' part too, by the block's first warp, which keeps to one launch the
// check that usually ends it.
template <typename T, int kThreads, bool kEntries>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(const __grid_constant__ Args a, int slices,
                                                                int slice_granules) {
  constexpr int kAhead = 4;
  extern __shared__ __align__(16) unsigned char smem[];
  if (a.unless_one && a.upstream[0] == 1.f) return;
  for (int64_t item = blockIdx.x; item < a.N * slices; item += gridDim.x) {
    const int64_t n = item / slices;
    const int slice = static_cast<int>(item % slices);
    const float m = a.stats[2 * n], sum = a.stats[2 * n + 1];
    T* grad = static_cast<T*>(a.grad) + n * a.grad_stride;
    const Granules<T> row(static_cast<const T*>(a.logits) + n * a.logits_stride, a.V), out(grad, a.V);
    if (sum == INFINITY) {  // no_row
      const int span = (out.count() + slices - 1) / slices;
      zero_granules(out, min(out.count(), slice * span), min(out.count(), (slice + 1) * span), kThreads, grad);
      continue;
    }
    const int lo = min(row.count(), slice * slice_granules), hi = min(row.count(), lo + slice_granules);
    const float coef = a.factor * a.upstream[n * a.upstream_stride] * (a.row_weight ? a.row_weight[n] : 1.f) * a.tau;
    const float mult = coef / sum;
    const bool same = row.phase == out.phase;
    for (int g0 = lo + threadIdx.x; g0 < hi; g0 += kAhead * kThreads) {
      uint4 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int g = g0 + u * kThreads;
        if (g >= hi) continue;
        if (row.whole(g))
          v[u] = *reinterpret_cast<const uint4*>(row.row + row.first(g));
        else
          v[u] = ragged(row, g);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int g = g0 + u * kThreads;
        if (g >= hi) continue;
        const uint4 o = grad_granule<T>(v[u], m, a.exp2_scale, mult);
        if (same && row.whole(g))
          *reinterpret_cast<uint4*>(grad + row.first(g)) = o;
        else
          store_elements<T>(o, row.first(g), row.V, grad);
      }
    }
    if constexpr (kEntries) {
      __syncthreads();  // the dense part is complete
      if (threadIdx.x < 32) {
        Entries e(smem, a.K, threadIdx.x);
        e.read(a, n);
        e.normalise(a);
        e.template finish<T, false>(a, row.row, m, 0.f);
        e.template store<T>(a, row.row, m, 1.f / sum, coef, grad);
      }
    }
  }
}

// What the entries add to long rows: the loss (kLoss), and the gradient of the logits that they name (a.grad set).
constexpr int kEntryWarps = 4;

template <typename T, bool kLoss>
__global__ void __launch_bounds__(kEntryWarps * 32) distill_entries_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kEntryWarps + warp;
  if (n >= a.N || (a.unless_one && a.upstream[0] == 1.f)) return;
  Entries e(smem + static_cast<size_t>(warp) * 12 * a.K, a.K, lane);
  const float weight = a.row_weight ? a.row_weight[n] : 1.f;
  const float2 st = reinterpret_cast<const float2*>(a.stats)[n];
  if (!e.read(a, n) || weight == 0.f) {
    if (kLoss && lane == 0) a.losses[n] = 0.f;
    return;
  }
  e.normalise(a);
  const T* row = static_cast<const T*>(a.logits) + n * a.logits_stride;
  const float loss = e.finish<T, kLoss>(a, row, st.x, logf(st.y));
  if (kLoss && lane == 0) a.losses[n] = weight * a.tau * loss;
  if (!a.grad) return;
  const float up = a.upstream ? a.upstream[n * a.upstream_stride] : 1.f;
  e.store<T>(a, row, st.x, 1.f / st.y, a.factor * up * weight * a.tau, static_cast<T*>(a.grad) + n * a.grad_stride);
}

// ------------------------------------------------------------------------------------------- rows of middling length

// A warp serves a row, all of it: no barrier stands between the readings, and a row of some KB is still in L1 or L2
// at its second one. kStats: find the statistics and the loss, else read the statistics.
constexpr int kMidWarps = 4;

template <typename T, bool kStats>
__global__ void __launch_bounds__(kMidWarps * 32) distill_warp_kernel(const __grid_constant__ Args a) {
  constexpr int kU = 4;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kMidWarps + warp;
  if (n >= a.N || (!kStats && a.unless_one && a.upstream[0] == 1.f)) return;
  Entries e(smem + static_cast<size_t>(warp) * 12 * a.K, a.K, lane);
  const float weight = a.row_weight ? a.row_weight[n] : 1.f;
  T* grad = a.grad ? static_cast<T*>(a.grad) + n * a.grad_stride : nullptr;
  if (!e.read(a, n) || weight == 0.f) {
    if (kStats && lane == 0) {
      a.losses[n] = 0.f;
      reinterpret_cast<float2*>(a.stats)[n] = no_row();
    }
    if (grad) {
      const Granules<T> out(grad, a.V);
      for (int g = lane; g < out.count(); g += 32) {
        if (out.whole(g))
          *reinterpret_cast<uint4*>(grad + out.first(g)) = make_uint4(0, 0, 0, 0);
        else
          store_elements<T>(make_uint4(0, 0, 0, 0), out.first(g), out.V, grad);
      }
    }
    return;
  }
  const Granules<T> row(static_cast<const T*>(a.logits) + n * a.logits_stride, a.V);
  // The whole granules [begin, end) go by vectors; the row's ragged ends, at most two, belong to lanes 0 and 1. A
  // lane past the last whole granule reads that one again and drops it: no branch stands between the loads.
  const int begin = row.first_whole(), end = row.end_whole();
  const int edge = row.ragged_end(lane);
  const uint4 ragged_end = edge >= 0 ? ragged(row, edge) : Granule<T>::none();
  auto load = [&](int g) { return *reinterpret_cast<const uint4*>(row.row + row.first(min(g, end - 1))); };
  float m, sum;
  if constexpr (kStats) {
    Stat st;
    auto add = [&](const uint4& most, auto&& terms) {
      const float top = warp_largest(Granule<T>::largest(most));
      if (top > st.m) {
        st.s *= exp2_approx((st.m - top) * a.exp2_scale);
        st.m = top;
      }
      st.s += terms(st.base());
    };
    add(ragged_end, [&](float base) { return exp2_sum<T>(ragged_end, base, a.exp2_scale); });
    for (int g0 = begin + lane; g0 < end + lane; g0 += kU * 32) {  // the same trips for all lanes
      uint4 v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) v[u] = load(g0 + u * 32);
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (g0 + u * 32 >= end) v[u] = Granule<T>::none();
      uint4 most = v[0];
#pragma unroll
      for (int u = 1; u < kU; ++u) most = Granule<T>::larger(most, v[u]);
      add(most, [&](float base) {
        float t = 0.f;
#pragma unroll
        for (int u = 0; u < kU; ++u) t += exp2_sum<T>(v[u], base, a.exp2_scale);
        return t;
      });
    }
    m = st.m;
    sum = lanes_sum<32>(st.s);
    if (m == -INFINITY) sum = NAN;  // a softmax over nothing
    if (lane == 0) reinterpret_cast<float2*>(a.stats)[n] = make_float2(m, sum);
  } else {
    m = a.stats[2 * n];
    sum = a.stats[2 * n + 1];
  }
  e.normalise(a);
  const float loss = e.finish<T, kStats>(a, row.row, m, logf(sum));
  if (kStats && lane == 0) a.losses[n] = weight * a.tau * loss;
  if (!grad) return;
  const float up = a.upstream ? a.upstream[n * a.upstream_stride] : 1.f;
  const float coef = a.factor * up * weight * a.tau, inv_sum = 1.f / sum, mult = coef * inv_sum;
  const bool same = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
  if (edge >= 0)
    store_elements<T>(grad_granule<T>(ragged_end, m, a.exp2_scale, mult), row.first(edge), row.V, grad);
  for (int g0 = begin + lane; g0 < end + lane; g0 += kU * 32) {
    uint4 v[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) v[u] = load(g0 + u * 32);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int g = g0 + u * 32;
      v[u] = grad_granule<T>(v[u], m, a.exp2_scale, mult);
      if (g >= end) continue;
      if (same)
        *reinterpret_cast<uint4*>(grad + row.first(g)) = v[u];
      else
        store_elements<T>(v[u], row.first(g), row.V, grad);
    }
  }
  __syncwarp();  // the dense pass is complete
  e.store<T>(a, row.row, m, inv_sum, coef, grad);
}

// total = factor * sum of the rows' losses, one block, a fixed order.
__global__ void __launch_bounds__(1024) total_kernel(int64_t N, float factor, const float* __restrict__ losses,
                                                     float* __restrict__ total) {
  __shared__ float red[32];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < N; i += 1024) s += losses[i];
  s = lanes_sum<32>(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = lanes_sum<32>(red[threadIdx.x]);
    if (threadIdx.x == 0) *total = factor * s;
  }
}

}  // namespace distill
}  // namespace ebr
