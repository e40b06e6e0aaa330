// key_sort.cuh: a stable sort of small integer keys with their positions, the common first step of the embedding's
// gradient (tokens by id) and of the expert route (slots by expert). Least-significant-digit counting passes of at
// most kMaxDigitBits bits: every key's place is  start of its digit + keys of that digit before it.
//
// Ranking inside a block: each warp owns a contiguous stretch of keys and walks it 32 at a time. __match_any_sync
// gives the lanes that hold the same digit, so a key's rank in its warp is the warp's running count of the digit plus
// the earlier lanes of the match; the counts of the block's warps are then scanned per digit. The order of equal keys
// never depends on timing, so everything built on it is deterministic.
//
// Bound by latency, not by bytes (a million bytes of ids): 162 slots take 4.5 us and 18,006 take 6.5 in one cluster,
// 124,416 take 6.9 in two kernels over the whole GPU, replayed from a CUDA graph.
#pragma once

#include <cooperative_groups.h>

#include "sm100.cuh"

namespace ebr {
namespace keysort {

constexpr int kMaxDigitBits = 10;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;

// The raw ids: int32 or int64, and every id outside [0, range) mapped to `range` (sorted last).
struct IdSource {
  const void* ids;
  int is64;
  int range;
  __device__ __forceinline__ int key(int64_t i) const {
    if (is64) {
      const int64_t v = static_cast<const int64_t*>(ids)[i];
      return v >= 0 && v < range ? static_cast<int>(v) : range;
    }
    const int v = static_cast<const int*>(ids)[i];
    return v >= 0 && v < range ? v : range;
  }
};

// One pass: keys and positions from (key_in, idx_in), or from the raw ids in their own order where key_in is NULL, to
// (key_out, idx_out).
struct Pass {
  const int* key_in;
  const int* idx_in;
  int* key_out;
  int* idx_out;
  int shift, bits;
};

// Where an expert route writes its last (only) pass: see include/ebr_tokens.h.
struct RouteOut {
  int* row_of;
  int* slot_of;
  int* offsets;
  int experts;
  int64_t capacity;
  int64_t rows;
};

// A small range that a sort's blocks zero on the way, this block's share of it. p is 16-byte aligned.
struct SmallZero {
  char* p;
  int64_t bytes;
  __device__ __forceinline__ void share(int part, int parts) const {
    const int64_t words = bytes / 16, step = static_cast<int64_t>(parts) * kSortThreads;
    for (int64_t i = static_cast<int64_t>(part) * kSortThreads + threadIdx.x; i < words; i += step)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
    if (part == 0 && threadIdx.x < bytes - words * 16) p[words * 16 + threadIdx.x] = 0;
  }
};

// ------------------------------------------------------------------------------------------------ block-level parts

// Ranks the block's keys [begin, begin + kItems * 32 of each warp) among the block's equal digits: dig / rank of item
// j of this thread (dig = -1 past the end), and after the call counts[w * digits + d] = keys of digit d in the warps
// before w, totals[d] = keys of digit d in the block. Keys with digit >= digits get no rank (dig = -1).
template <int kItems, typename KeyFn>
__device__ __forceinline__ void rank_block(int64_t warp_begin, int64_t warp_end, int digits, KeyFn key_of,
                                           uint16_t* counts, int* totals, int (&dig)[kItems], int (&rank)[kItems]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < digits * kSortWarps; i += kSortThreads) counts[i] = 0;
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = warp_begin + j * 32 + lane;
    dig[j] = i < warp_end ? key_of(i, j) : -1;
    if (dig[j] >= digits) dig[j] = -1;
  }
  __syncthreads();
  uint16_t* mine = counts + warp * digits;
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const unsigned peers = __match_any_sync(0xffffffffu, dig[j]);
    const unsigned before = peers & ((1u << lane) - 1u);
    rank[j] = 0;
    if (dig[j] >= 0) rank[j] = mine[dig[j]] + __popc(before);
    __syncwarp();
    if (dig[j] >= 0 && before == 0) mine[dig[j]] = static_cast<uint16_t>(mine[dig[j]] + __popc(peers));
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) {
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = counts[w * digits + d];
      counts[w * digits + d] = static_cast<uint16_t>(run);
      run += c;
    }
    totals[d] = run;
  }
  __syncthreads();
}

// Exclusive sum over the block of one value per thread (thread order). `warp_sums` holds kSortWarps ints.
__device__ __forceinline__ int block_exclusive(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // warp_sums may still be read by an earlier call
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    const int s = warp_sums[lane];
    int t = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += y;
    }
    warp_sums[lane] = t - s;
    if (lane == 31) *total = t;
  }
  __syncthreads();
  return x - v + warp_sums[warp];
}

// Rows of no slot, and the offsets: the part of a route that does not depend on single slots. digit_start /
// digit_total [experts] are shared arrays; `part` of `parts` blocks share the row walk.
__device__ __forceinline__ void finish_route(const RouteOut& r, const int* digit_start, const int* digit_total,
                                             int live, int part, int parts) {
  if (part == 0) {
    for (int e = threadIdx.x; e < r.experts; e += kSortThreads) r.offsets[e] = digit_start[e];
    if (threadIdx.x == 0) r.offsets[r.experts] = live;
  }
  const int64_t first = r.capacity ? 0 : live;
  for (int64_t row = first + static_cast<int64_t>(part) * kSortThreads + threadIdx.x; row < r.rows;
       row += static_cast<int64_t>(parts) * kSortThreads) {
    if (r.capacity) {
      const int64_t e = row / r.capacity;
      if (row - e * r.capacity < digit_total[e]) continue;
    }
    r.slot_of[row] = -1;
  }
}

__device__ __forceinline__ void put_slot(const RouteOut& r, int slot, int e, int place, int start) {
  int64_t row = place;
  if (r.capacity) {
    const int64_t in = place - start;
    row = in < r.capacity ? e * r.capacity + in : -1;
  }
  r.row_of[slot] = static_cast<int>(row);
  if (row >= 0) r.slot_of[row] = slot;
}

// ------------------------------------------------------------------------------------------------ one cluster

// The whole sort, all its passes, in one cluster of up to 16 CTAs: a pass's digit totals are exchanged through
// distributed shared memory, and its output (a scratch array, which stays in L2) is read by the next pass after a
// cluster barrier. One launch: at some thousand keys the launches, not the keys, are the cost.
struct ClusterSort {
  IdSource src;
  int64_t n;
  int passes;
  Pass pass[3];
  RouteOut route;  // row_of != NULL: an expert route (one pass)
  SmallZero zero;
};

// What a kernel that may run beside its predecessor in the stream says, and what it waits with.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Zeros a byte range, kZeroPiece bytes to a block (contiguous pieces: 7.1 TB/s on 537 MB; a grid-stride walk 5.9). It
// is launched behind the cluster sort, which does not touch the range, to run beside it on the SMs that the sort
// leaves free; the last block ends only after the sort, so whatever follows in the stream finds both done.
constexpr int64_t kZeroPiece = 128 * 1024;

__global__ void __launch_bounds__(1024) zero_kernel(char* p, int64_t bytes) {
  const int64_t begin = blockIdx.x * kZeroPiece, end = min(bytes, begin + kZeroPiece);
  const int64_t words = (end - begin) / 16;  // p is 16-byte aligned
  uint4* w = reinterpret_cast<uint4*>(p + begin);
  for (int64_t i = threadIdx.x; i < words; i += 1024) w[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = begin + words * 16 + threadIdx.x; i < end; i += 1024) p[i] = 0;
  if (blockIdx.x == gridDim.x - 1) wait_for_previous();
}

inline size_t cluster_sort_smem(int bits) {
  const size_t digits = size_t{1} << bits;
  return digits * kSortWarps * sizeof(uint16_t) + 3 * digits * sizeof(int) + (kSortWarps + 4) * sizeof(int);
}

template <int kItems>
__global__ void __launch_bounds__(kSortThreads, 1) cluster_sort_kernel(const __grid_constant__ ClusterSort a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks());
  const int me = static_cast<int>(cluster.block_rank());
  let_next_start();
  a.zero.share(me, ctas);
  extern __shared__ __align__(16) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t per_cta = (a.n + ctas - 1) / ctas;
  const int64_t cta_end = min(a.n, (me + 1) * per_cta);
  const int64_t warp_begin = me * per_cta + static_cast<int64_t>(warp) * (kItems * 32);
  const int64_t warp_end = min(cta_end, warp_begin + kItems * 32);
  for (int p = 0; p < a.passes; ++p) {
    const Pass ps = a.pass[p];
    const bool route = a.route.row_of != nullptr;
    const int digits = route ? a.route.experts : 1 << ps.bits;
    uint16_t* counts = reinterpret_cast<uint16_t*>(smem);
    int* totals = reinterpret_cast<int*>(smem + (static_cast<size_t>(1) << ps.bits) * kSortWarps * sizeof(uint16_t));
    int* start = totals + (1 << ps.bits);  // first place of this CTA's keys of a digit
    int* dstart = start + (1 << ps.bits);  // first place of a digit's keys
    int* warp_sums = dstart + (1 << ps.bits);
    int* live = warp_sums + kSortWarps;
    int key[kItems], dig[kItems], rank[kItems];
    rank_block<kItems>(
        warp_begin, warp_end, digits,
        [&](int64_t i, int j) {
          key[j] = ps.key_in ? __ldcg(ps.key_in + i) : a.src.key(i);
          return route ? key[j] : (key[j] >> ps.shift) & (digits - 1);
        },
        counts, totals, dig, rank);
    cluster.sync();
    int all = 0, before = 0;
    const int d = threadIdx.x;  // digits <= kSortThreads
    if (d < digits) {
      for (int c = 0; c < ctas; ++c) {
        const int t = *cluster.map_shared_rank(totals + d, c);
        if (c < me) before += t;
        all += t;
      }
    }
    const int first = block_exclusive(all, warp_sums, live);
    if (d < digits) {
      start[d] = first + before;
      dstart[d] = first;
    }
    cluster.sync();  // totals have been read everywhere; start / dstart are complete in this CTA
    if (route) {
#pragma unroll
      for (int j = 0; j < kItems; ++j) {
        const int64_t i = warp_begin + j * 32 + lane;
        if (i >= warp_end) continue;
        if (dig[j] < 0)
          a.route.row_of[i] = -1;
        else
          put_slot(a.route, static_cast<int>(i), dig[j], start[dig[j]] + counts[warp * digits + dig[j]] + rank[j],
                   dstart[dig[j]]);
      }
      __syncthreads();
      if (d < digits) start[d] = all;
      __syncthreads();
      finish_route(a.route, dstart, start, *live, me, ctas);
      return;
    }
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      if (dig[j] < 0) continue;
      const int64_t i = warp_begin + j * 32 + lane;
      const int place = start[dig[j]] + counts[warp * digits + dig[j]] + rank[j];
      ps.key_out[place] = key[j];
      ps.idx_out[place] = ps.idx_in ? __ldcg(ps.idx_in + i) : static_cast<int>(i);
    }
    if (p + 1 < a.passes) {
      __threadfence();
      cluster.sync();
    }
  }
}

// ------------------------------------------------------------------------------------------------ whole grid

// For more keys: per pass, one block per tile of kSortThreads * kItems keys counts its digits, and one block per tile
// ranks and places its keys. With up to kMaxTiles tiles the second kernel adds up the tiles before its own itself;
// with more, a kernel between the two scans the counts.
constexpr int kMaxTiles = 256;

struct GridSort {
  IdSource src;
  int64_t n;
  Pass pass;
  int digits;
  int tiles;
  int scanned;  // counts hold the sums over the tiles before, totals the sums over all
  int* counts;  // [tiles][digits]
  int* totals;  // [digits], where scanned
  RouteOut route;
  SmallZero zero;  // of the first pass
};

__device__ __forceinline__ int grid_digit(const GridSort& a, int key) {
  return a.route.row_of ? key : (key >> a.pass.shift) & (a.digits - 1);
}

template <int kItems>
__global__ void __launch_bounds__(kSortThreads) grid_count_kernel(const __grid_constant__ GridSort a) {
  __shared__ int hist[1 << kMaxDigitBits];
  if (!a.pass.key_in) a.zero.share(blockIdx.x, gridDim.x);
  for (int d = threadIdx.x; d < a.digits; d += kSortThreads) hist[d] = 0;
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * kSortThreads * kItems;
  int dig[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = begin + j * kSortThreads + threadIdx.x;
    dig[j] = i < a.n ? grid_digit(a, a.pass.key_in ? a.pass.key_in[i] : a.src.key(i)) : a.digits;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j)
    if (dig[j] < a.digits) atomicAdd(&hist[dig[j]], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < a.digits; d += kSortThreads)
    a.counts[static_cast<int64_t>(blockIdx.x) * a.digits + d] = hist[d];
}

__global__ void __launch_bounds__(kSortThreads) grid_scan_kernel(const __grid_constant__ GridSort a) {
  __shared__ int warp_sums[kSortWarps];
  __shared__ int chunk_total;
  int* column = a.counts + blockIdx.x;
  int run = 0;
  for (int t0 = 0; t0 < a.tiles; t0 += kSortThreads) {
    const int t = t0 + threadIdx.x;
    const int v = t < a.tiles ? column[static_cast<int64_t>(t) * a.digits] : 0;
    const int ex = block_exclusive(v, warp_sums, &chunk_total);
    if (t < a.tiles) column[static_cast<int64_t>(t) * a.digits] = run + ex;
    run += chunk_total;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.totals[blockIdx.x] = run;
}

template <int kItems>
__global__ void __launch_bounds__(kSortThreads) grid_place_kernel(const __grid_constant__ GridSort a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int digits = a.digits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint16_t* counts = reinterpret_cast<uint16_t*>(smem);
  int* totals = reinterpret_cast<int*>(smem + static_cast<size_t>((digits + 1) & ~1) * kSortWarps * sizeof(uint16_t));
  int* start = totals + digits;
  int* dstart = start + digits;
  int* warp_sums = dstart + digits;
  int* live = warp_sums + kSortWarps;
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * kSortThreads * kItems;
  const int64_t end = min(a.n, begin + kSortThreads * kItems);
  const int64_t warp_begin = begin + static_cast<int64_t>(warp) * (kItems * 32);
  const int64_t warp_end = min(end, warp_begin + kItems * 32);
  int key[kItems], dig[kItems], rank[kItems];
  rank_block<kItems>(
      warp_begin, warp_end, digits,
      [&](int64_t i, int j) {
        key[j] = a.pass.key_in ? a.pass.key_in[i] : a.src.key(i);
        return grid_digit(a, key[j]);
      },
      counts, totals, dig, rank);
  const int d = threadIdx.x;
  if (d < digits) {
    totals[d] = a.scanned ? a.totals[d] : 0;
    start[d] = a.scanned ? a.counts[static_cast<int64_t>(blockIdx.x) * digits + d] : 0;
  }
  __syncthreads();
  if (!a.scanned) {  // sums over the tiles: `groups` threads share a digit
    int wide = 1;
    while (wide < digits) wide *= 2;
    const int groups = kSortThreads / wide, mine = threadIdx.x & (wide - 1);
    if (mine < digits) {
      int before = 0, all = 0;
#pragma unroll 8
      for (int t = threadIdx.x / wide; t < a.tiles; t += groups) {
        const int c = a.counts[static_cast<int64_t>(t) * digits + mine];
        all += c;
        if (t < static_cast<int>(blockIdx.x)) before += c;
      }
      atomicAdd(&totals[mine], all);
      atomicAdd(&start[mine], before);
    }
    __syncthreads();
  }
  const int first = block_exclusive(d < digits ? totals[d] : 0, warp_sums, live);
  if (d < digits) {
    dstart[d] = first;
    start[d] += first;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = warp_begin + j * 32 + lane;
    if (i >= warp_end) continue;
    if (dig[j] < 0) {
      if (a.route.row_of) a.route.row_of[i] = -1;
      continue;
    }
    const int place = start[dig[j]] + counts[warp * digits + dig[j]] + rank[j];
    if (a.route.row_of) {
      put_slot(a.route, static_cast<int>(i), dig[j], place, dstart[dig[j]]);
    } else {
      a.pass.key_out[place] = key[j];
      a.pass.idx_out[place] = a.pass.idx_in ? a.pass.idx_in[i] : static_cast<int>(i);
    }
  }
  if (a.route.row_of) finish_route(a.route, dstart, totals, *live, blockIdx.x, gridDim.x);
}

inline size_t grid_place_smem(int digits) {
  return static_cast<size_t>((digits + 1) & ~1) * kSortWarps * sizeof(uint16_t) + 3 * digits * sizeof(int) +
         (kSortWarps + 4) * sizeof(int);
}

}  // namespace keysort
}  // namespace ebr
