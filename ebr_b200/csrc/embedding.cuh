// embedding.cuh: the scaled embedding out[t] = scale * W[id_t] and its gradient dW[v] = scale * sum_{t: id_t = v} g[t].
//
// Both are bound by HBM: the lookup writes n rows (and reads the distinct rows of W), the gradient reads n rows of g
// and writes the whole table. The gradient needs no atomics: the tokens are sorted by id (key_sort.cuh), so the rows of
// one id are neighbours in the sorted order. The sorted tokens are cut into chunks of R rows; a warp sums the runs of
// equal ids of its chunk for 32 vectors of columns. A run that lies in one chunk goes straight to dW; a run that crosses
// chunks leaves one float32 partial sum per chunk, which a second kernel adds in chunk order. A table of ten rows
// under 62,208 tokens (runs of thousands) and one of 131,072 rows (runs of one or two) take the same path.
#pragma once

#include "key_sort.cuh"
#include "layers.cuh"

namespace ebr {
namespace embed {

using keysort::IdSource;

// V consecutive elements as floats, in accesses of at most 16 bytes.
template <typename T, int V>
__device__ __forceinline__ void load_f(const T* p, float (&out)[V]) {
  constexpr int kStep = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
#pragma unroll
  for (int s = 0; s < V; s += kStep) {
    const layers::Pack<T, kStep> pk = *reinterpret_cast<const layers::Pack<T, kStep>*>(p + s);
#pragma unroll
    for (int i = 0; i < kStep; ++i) out[s + i] = Elem<T>::load(&pk.e[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_f(T* p, const float (&in)[V]) {
  constexpr int kStep = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
#pragma unroll
  for (int s = 0; s < V; s += kStep) {
    layers::Pack<T, kStep> pk;
#pragma unroll
    for (int i = 0; i < kStep; ++i) pk.e[i] = Elem<T>::to(in[s + i]);
    *reinterpret_cast<layers::Pack<T, kStep>*>(p + s) = pk;
  }
}

// ------------------------------------------------------------------------------------------------ lookup

// A warp writes one token's 32 vectors of columns (blockIdx.y picks them); kRows tokens' loads are in flight at once.
constexpr int kLookupWarps = 8, kLookupRows = 4;

template <typename TW, typename TO, int V>
__global__ void __launch_bounds__(kLookupWarps * 32) lookup_kernel(IdSource src, int64_t n, int64_t C, float scale,
                                                                   const TW* __restrict__ w, int64_t w_stride,
                                                                   TO* __restrict__ out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (static_cast<int64_t>(blockIdx.y) * 32 + lane) * V;
  if (c >= C) return;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kLookupWarps;
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * kLookupWarps + warp; t0 < n; t0 += step * kLookupRows) {
    float v[kLookupRows][V];
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
      const int64_t t = t0 + u * step;
      const int id = t < n ? src.key(t) : src.range;
      if (id < src.range) {
        load_f<TW, V>(w + id * w_stride + c, v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[u][i] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
      const int64_t t = t0 + u * step;
      if (t >= n) break;
#pragma unroll
      for (int i = 0; i < V; ++i) v[u][i] *= scale;
      store_f<TO, V>(out + t * C + c, v[u]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ gradient

constexpr int kGradWarps = 8;

// part[chunk][0]: the sum of the run that the chunk starts in the middle of; part[chunk][1]: of the run that starts in
// the chunk and goes on in the next. Rows of C floats.
template <typename TG, typename TW, int V>
__global__ void __launch_bounds__(kGradWarps * 32) grad_chunk_kernel(int n, int range, int64_t C, int R,
                                                                     const int* __restrict__ key,
                                                                     const int* __restrict__ order,
                                                                     const TG* __restrict__ g, int64_t g_stride,
                                                                     float scale, TW* __restrict__ dw,
                                                                     float* __restrict__ part) {
  constexpr int kAhead = 8;  // rows in flight
  const int lane = threadIdx.x & 31;
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) * kGradWarps + (threadIdx.x >> 5);
  const int64_t begin = chunk * R;
  if (begin >= n) return;
  const int64_t end = min(static_cast<int64_t>(n), begin + R);
  const int64_t c = (static_cast<int64_t>(blockIdx.y) * 32 + lane) * V;
  const bool live = c < C;
  int cur = key[begin];
  if (cur >= range) return;  // only ids of no table row from here on
  bool head = begin > 0 && key[begin - 1] == cur;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  auto flush = [&](bool goes_on) {
    if (!live) return;
    if (head || goes_on) {
      store_f<float, V>(part + (chunk * 2 + (head ? 0 : 1)) * C + c, acc);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= scale;
      store_f<TW, V>(dw + cur * C + c, acc);
    }
  };
  for (int64_t r0 = begin; r0 < end; r0 += 32) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(32), end - r0));
    const int my_key = lane < rows ? key[r0 + lane] : range;
    const int my_row = lane < rows ? order[r0 + lane] : 0;
    for (int j0 = 0; j0 < rows; j0 += kAhead) {
      float v[kAhead][V];
      int k[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = j0 + u;
        k[u] = __shfl_sync(0xffffffffu, my_key, j & 31);
        const int64_t row = __shfl_sync(0xffffffffu, my_row, j & 31);
        if (j < rows && k[u] < range && live) {
          load_f<TG, V>(g + row * g_stride + c, v[u]);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) v[u][i] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (j0 + u >= rows) break;
        if (k[u] != cur) {
          flush(false);
          if (k[u] >= range) return;
          cur = k[u];
          head = false;
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += v[u][i];
      }
    }
  }
  flush(end < n && key[end] == cur);
}

// Runs that cross chunks: a block looks at kJoinChunks chunk ends; where the run at a chunk's end started in that chunk
// and goes on, the block adds its partials in chunk order (its warps take every kJoinWarps-th partial) for 32 vectors of
// four columns.
constexpr int kJoinWarps = 8, kJoinChunks = 32;

template <typename TW>
__global__ void __launch_bounds__(kJoinWarps * 32) grad_join_kernel(int n, int range, int64_t C, int R, int chunks,
                                                                    const int* __restrict__ key, float scale,
                                                                    TW* __restrict__ dw,
                                                                    const float* __restrict__ part) {
  __shared__ float4 sums[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kJoinChunks;
  bool owner = false;
  int id = 0;
  if (first + lane < chunks) {
    const int64_t begin = (first + lane) * R, end = begin + R;
    if (end < n) {
      id = key[end - 1];
      owner = id < range && key[end] == id && (begin == 0 || key[begin - 1] != id);
    }
  }
  unsigned owners = __ballot_sync(0xffffffffu, owner);
  const int64_t c = (static_cast<int64_t>(blockIdx.y) * 32 + lane) * 4;
  while (owners) {
    const int o = __ffs(owners) - 1;
    owners &= owners - 1;
    const int64_t chunk = first + o;
    const int k = __shfl_sync(0xffffffffu, id, o);
    // the last chunk that starts with this id: the keys at the chunks' starts are in order
    int64_t lo = chunk + 1, hi = chunks - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) / 2;
      if (key[mid * R] == k) lo = mid; else hi = mid - 1;
    }
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int64_t j = chunk + warp; j <= lo; j += kJoinWarps) {
      const float* p = part + (j * 2 + (j == chunk ? 1 : 0)) * C;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < C) (&s.x)[i] += p[c + i];
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int w = 1; w < kJoinWarps; ++w) {
        const float4 t = sums[w][lane];
        s.x += t.x;
        s.y += t.y;
        s.z += t.z;
        s.w += t.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < C) dw[k * C + c + i] = Elem<TW>::to((&s.x)[i] * scale);
    }
    __syncthreads();
  }
}

}  // namespace embed
}  // namespace ebr
