// embedding.cuh: the scaled embedding out[t] = scale * W[id_t] and its gradient dW[v] = scale * sum_{t: id_t = v}
// g[t].
//
// Both are bound by HBM: the lookup writes n rows (and reads the distinct rows of W), the gradient reads n rows of g
// and writes the whole table. The gradient needs no atomics: the tokens are sorted by id (key_sort.cuh), so the rows
// of one id are neighbours in the sorted order. The sorted tokens are cut into chunks of R rows; a warp sums the runs
// of equal ids of its chunk for 32 vectors of columns. A run that lies in one chunk goes straight to dW; a run that
// crosses chunks leaves one float32 partial sum per chunk, which a second kernel adds in chunk order. A table of ten
// rows under 62,208 tokens (runs of thousands) and one of 131,072 rows (runs of one or two) take the same path.
//
// Measured, replayed from a CUDA graph (warm: one after another; cold: behind a flush of L2): the lookup of 16,384
// bfloat16 tokens of 2,048 columns 16.5 us warm (8.1 TB/s of its rows and output, some of it from L2), of 62,208 board
// tokens of 512 columns from a float32 table 16.4 us warm and 20.5 cold (3.9 and 3.1 TB/s: the latency of a single
// wave of 3,900 warps with four rows in flight each; issue slots 41 %, resident warps 38 %); the gradients of the same
// 111 us warm (5.5 TB/s; 74 of it zero the table, beside the sort) and 27 us warm, 39 to 41 cold (the latency of four
// short kernels: two of the sort, chunks, join). Rows of an odd number of 16-bit elements go two bytes a lane: 30,000
// tokens of 1,001 bfloat16 of a table of 50,000 take 31 us (lookup) and 86 (gradient) warm, of 1,000 columns 21 and 53.
#pragma once

#include <type_traits>

#include "key_sort.cuh"
#include "layers.cuh"

namespace ebr {
namespace embed {

using keysort::IdSource;

// kBytes bytes as one access.
template <int kBytes>
struct Word;
template <>
struct Word<2> {
  using type = unsigned short;
};
template <>
struct Word<4> {
  using type = unsigned;
};
template <>
struct Word<8> {
  using type = uint2;
};
template <>
struct Word<16> {
  using type = uint4;
};

// V elements of T as they are in memory (at most 16 bytes), and as floats. The 16-bit types are converted two at a
// time from whole words.
template <typename T, int V>
struct Raw {
  using W = typename Word<V * sizeof(T)>::type;
  W w = {};
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
  __device__ __forceinline__ void widen(float (&v)[V]) const {
    if constexpr (sizeof(T) == 4) {
      const float* f = reinterpret_cast<const float*>(&w);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = f[i];
    } else if constexpr (V == 1) {
      v[0] = Elem<T>::load(reinterpret_cast<const T*>(&w));
    } else {
      const unsigned* u = reinterpret_cast<const unsigned*>(&w);
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          v[i] = __uint_as_float(u[i / 2] << 16);
          v[i + 1] = __uint_as_float(u[i / 2] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i / 2]));
          v[i] = f.x;
          v[i + 1] = f.y;
        }
      }
    }
  }
  __device__ __forceinline__ void narrow(const float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
      float* f = reinterpret_cast<float*>(&w);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = v[i];
    } else if constexpr (V == 1) {
      *reinterpret_cast<T*>(&w) = Elem<T>::to(v[0]);
    } else {
      unsigned* u = reinterpret_cast<unsigned*>(&w);
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float2 f = make_float2(v[i], v[i + 1]);
        if constexpr (std::is_same_v<T, __nv_bfloat16>)
          *reinterpret_cast<__nv_bfloat162*>(&u[i / 2]) = __float22bfloat162_rn(f);
        else
          *reinterpret_cast<__half2*>(&u[i / 2]) = __float22half2_rn(f);
      }
    }
  }
};

// V consecutive elements as floats, in accesses of at most 16 bytes.
template <typename T, int V>
__device__ __forceinline__ void load_f(const T* p, float (&out)[V]) {
  constexpr int kStep = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
#pragma unroll
  for (int s = 0; s < V; s += kStep) {
    Raw<T, kStep> r;
    r.load(p + s);
    r.widen(*reinterpret_cast<float(*)[kStep]>(out + s));
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_f(T* p, const float (&in)[V]) {
  constexpr int kStep = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
#pragma unroll
  for (int s = 0; s < V; s += kStep) {
    Raw<T, kStep> r;
    r.narrow(*reinterpret_cast<const float(*)[kStep]>(in + s));
    r.store(p + s);
  }
}

// ------------------------------------------------------------------------------------------------ lookup

// A warp writes up to 32 consecutive tokens' parts of kU * 32 vectors of columns (blockIdx.y picks them): its lanes
// read the ids at once, and kLookupAhead / kU rows are in flight, so that the chain id -> row -> store is paid once
// for many rows. Whole rows by one warp where they fit: neighbouring rows are then written as one stretch.
constexpr int kLookupWarps = 4, kLookupAhead = 4;

template <typename TW, typename TO, int V, int kU>
__global__ void __launch_bounds__(kLookupWarps * 32) lookup_kernel(IdSource src, int64_t n, int64_t C, float scale,
                                                                   const TW* __restrict__ w, int64_t w_stride,
                                                                   TO* __restrict__ out, int per_warp) {
  constexpr int kRows = kLookupAhead / kU;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c0 = (static_cast<int64_t>(blockIdx.y) * kU * 32 + lane) * V;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kLookupWarps + warp) * per_warp;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(per_warp), n - t0));  // may be <= 0
  const int my_id = lane < tokens ? src.key(t0 + lane) : src.range;
  TO* dst = out + t0 * C + c0;
  for (int j0 = 0; j0 < tokens; j0 += kRows) {
    float v[kRows][kU][V];
    int id[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      // Lanes past the row and ids of no row read somewhere valid: no branch stands between the loads.
      id[r] = __shfl_sync(0xffffffffu, my_id, (j0 + r) & 31);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int64_t c = c0 + u * 32 * V;
        load_f<TW, V>(w + (id[r] < src.range ? id[r] : 0) * w_stride + (c < C ? c : 0), v[r][u]);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (j0 + r >= tokens || c0 + u * 32 * V >= C) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) v[r][u][i] = id[r] < src.range ? v[r][u][i] * scale : 0.f;
        store_f<TO, V>(dst + (j0 + r) * C + u * 32 * V, v[r][u]);
      }
  }
}

// ------------------------------------------------------------------------------------------------ gradient

constexpr int kGradWarps = 8;

// part[chunk][0]: the sum of the run that the chunk starts in the middle of; part[chunk][1]: of the run that starts
// in the chunk and goes on in the next. Rows of C floats.
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
  auto add = [&](const Raw<TG, V>& r) {
    float v[V];
    r.widen(v);
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += v[i];
  };
  auto flush = [&](bool goes_on) {
    if (live) {
      if (head || goes_on) {
        store_f<float, V>(part + (chunk * 2 + (head ? 0 : 1)) * C + c, acc);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] *= scale;
        store_f<TW, V>(dw + cur * C + c, acc);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    head = false;
  };
  for (int64_t r0 = begin; r0 < end; r0 += 32) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(32), end - r0));
    const int my_key = lane < rows ? key[r0 + lane] : range;
    const int my_row = lane < rows ? order[r0 + lane] : 0;
    const int valid = __popc(__ballot_sync(0xffffffffu, my_key < range));  // the first ones: the keys are sorted
    for (int j0 = 0; j0 < valid; j0 += kAhead) {
      Raw<TG, V> v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        // Lanes past the row and rows past the last read somewhere valid: no branch stands between the loads.
        const int64_t row = __shfl_sync(0xffffffffu, my_row, (j0 + u) & 31);
        v[u].load(g + row * g_stride + (live ? c : 0));
      }
      const int last = __shfl_sync(0xffffffffu, my_key, min(j0 + kAhead, valid) - 1);
      if (last == cur && j0 + kAhead <= valid) {  // one run
#pragma unroll
        for (int u = 0; u < kAhead; ++u) add(v[u]);
      } else {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int k = __shfl_sync(0xffffffffu, my_key, (j0 + u) & 31);
          if (j0 + u >= valid) continue;
          if (k != cur) {
            flush(false);
            cur = k;
          }
          add(v[u]);
        }
      }
    }
    if (valid < rows) {  // the rest of the chunk, and all behind it, has ids of no table row
      flush(false);
      return;
    }
  }
  flush(end < n && key[end] == cur);
}

// Runs that cross chunks. A block looks at the ends of kJoinChunks chunks, a warp at one of them: where the run at a
// chunk's end started in that chunk and goes on, its partials are added in chunk order. A run of a few chunks is
// added by its warp, 32 vectors of four columns; a long one by the whole block, every warp taking every kJoinWarps-th
// partial.
constexpr int kJoinWarps = 32, kJoinChunks = 32, kJoinShort = 16;

template <typename TW>
__global__ void __launch_bounds__(kJoinWarps * 32) grad_join_kernel(int n, int range, int64_t C, int R, int chunks,
                                                                    const int* __restrict__ key, float scale,
                                                                    TW* __restrict__ dw,
                                                                    const float* __restrict__ part) {
  constexpr int kAhead = 8;
  __shared__ float4 sums[kJoinWarps][32];
  __shared__ int ids[kJoinChunks];
  __shared__ int lasts[kJoinChunks];  // the last chunk of a long run, or -1
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kJoinChunks;
  const int64_t c = (static_cast<int64_t>(blockIdx.y) * 32 + lane) * 4;
  const bool whole = C % 4 == 0;
  // the partials of chunks from, from + step, ... up to `last` of the run that starts in `owner`
  auto gather = [&](int64_t owner, int64_t from, int64_t last, int step) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < C)
      for (int64_t j0 = from; j0 <= last; j0 += kAhead * step) {
        float4 v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int64_t j = j0 + u * step;
          v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (j > last) continue;
          const float* p = part + (j * 2 + (j == owner ? 1 : 0)) * C + c;
          if (whole) {
            v[u] = *reinterpret_cast<const float4*>(p);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c + i < C) (&v[u].x)[i] = p[i];
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          s.x += v[u].x;
          s.y += v[u].y;
          s.z += v[u].z;
          s.w += v[u].w;
        }
      }
    return s;
  };
  auto put = [&](int id, const float4& s) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < C) dw[id * C + c + i] = Elem<TW>::to((&s.x)[i] * scale);
  };
  {
    const int64_t chunk = first + warp, begin = chunk * R, end = begin + R;
    int id = -1;
    int64_t last = -1;
    if (chunk < chunks && end < n) {
      id = key[end - 1];
      if (id >= range || key[end] != id || (begin > 0 && key[begin - 1] == id)) id = -1;
    }
    if (id >= 0) {  // the last chunk that starts with this id: the keys at the chunks' starts are in order
      // [lo, hi]; 32 probes at a time
      int64_t lo = chunk + 1, hi = chunks - 1;
      while (lo < hi) {
        const int64_t gap = (hi - lo + 31) / 32, at = min(hi, lo + (lane + 1) * gap);
        const int hits = __popc(__ballot_sync(0xffffffffu, key[at * R] == id));  // the first ones
        hi = min(hi, lo + (hits + 1) * gap - 1);
        lo = min(hi, lo + hits * gap);
      }
      last = lo;
      if (last - chunk < kJoinShort) {
        put(id, gather(chunk, chunk, last, 1));
        last = -1;
      }
    }
    if (lane == 0) {
      ids[warp] = id;
      lasts[warp] = static_cast<int>(last);
    }
  }
  __syncthreads();
  for (int o = 0; o < kJoinChunks; ++o) {
    if (lasts[o] < 0) continue;
    const int64_t chunk = first + o;
    float4 s = gather(chunk, chunk + warp, lasts[o], kJoinWarps);
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0) {
#pragma unroll 8
      for (int w = 1; w < kJoinWarps; ++w) {
        const float4 t = sums[w][lane];
        s.x += t.x;
        s.y += t.y;
        s.z += t.z;
        s.w += t.w;
      }
      put(ids[o], s);
    }
    __syncthreads();
  }
}

// Few tokens: kShare warps own a table row's part and go through all ids themselves, each through its stretch of
// them, adding the rows of their own in their order. No sort, no zeroing, no joining: one launch, where the launches
// are the cost.
template <typename TG, typename TW, int V, int kShare>
__global__ void __launch_bounds__(kGradWarps * 32) grad_few_kernel(IdSource src, int n, int64_t C,
                                                                   const TG* __restrict__ g, int64_t g_stride,
                                                                   float scale, TW* __restrict__ dw) {
  constexpr int kAhead = 8, kOwners = kGradWarps / kShare;
  __shared__ float sums[kShare > 1 ? kGradWarps : 1][32][V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % kShare;
  const int64_t v = static_cast<int64_t>(blockIdx.x) * kOwners + warp / kShare;
  if (kShare == 1 && v >= src.range) return;
  const int64_t c = (static_cast<int64_t>(blockIdx.y) * 32 + lane) * V;
  const int span = ((n + kShare - 1) / kShare + 31) / 32 * 32, end = min(n, (part + 1) * span);
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  for (int t0 = part * span; t0 < end; t0 += 32) {
    unsigned mine = __ballot_sync(0xffffffffu, t0 + lane < end && src.key(t0 + lane) == v);
    if (v >= src.range) mine = 0;
    while (mine) {
      Raw<TG, V> r[kAhead];
      unsigned left = mine;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {  // past the last one: the first again, not used
        r[u].load(g + (t0 + __ffs(left ? left : mine) - 1) * g_stride + (c < C ? c : 0));
        left &= left - 1;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (!mine) break;
        float x[V];
        r[u].widen(x);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += x[i];
        mine &= mine - 1;
      }
    }
  }
  if constexpr (kShare > 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) sums[warp][lane][i] = acc[i];
    __syncthreads();
    if (part > 0 || v >= src.range) return;
#pragma unroll
    for (int p = 1; p < kShare; ++p)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += sums[warp + p][lane][i];
  }
  if (c >= C) return;
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] *= scale;
  store_f<TW, V>(dw + v * C + c, acc);
}

}  // namespace embed
}  // namespace ebr
