// tokens_capi.cuh: the C ABI of include/ebr_tokens.h (included at the end of capi.cu, after layers_capi.cuh, whose
// dtype and alignment helpers it uses). Validates arguments, picks the access width and launch shape, and launches
// the kernels of key_sort.cuh, embedding.cuh, experts.cuh and distill.cuh on the caller's stream.
#pragma once

#include "../../include/ebr_tokens.h"
#include "distill.cuh"
#include "embedding.cuh"
#include "experts.cuh"
#include "key_sort.cuh"

namespace {

using ebr::keysort::ClusterSort;
using ebr::keysort::GridSort;
using ebr::keysort::IdSource;

constexpr int64_t kMaxSortKeys = int64_t{1} << 30;
constexpr int kMaxExperts = 1 << ebr::keysort::kMaxDigitBits;

int check_id_type(int id_type) {
  return id_type == EBR_INT32 || id_type == EBR_INT64 ? EBR_OK : set_error(EBR_ERR_DTYPE, "ids must be int32 or int64%s%s");
}

// Whether p starts where an element of `size` bytes may.
bool on_boundary(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

int check_ids(const void* ids, int id_type) {
  return on_boundary(ids, id_type == EBR_INT64 ? 8 : 4) ? EBR_OK : set_error(EBR_ERR_STRIDE, "unaligned ids%s%s");
}

// Arrays that start where none of their elements may are refused here: in a kernel they would be a fault.
struct Array {
  const void* p;
  size_t size;
};

int check_arrays(std::initializer_list<Array> arrays) {
  for (const Array& a : arrays)
    if (!on_boundary(a.p, a.size)) return set_error(EBR_ERR_STRIDE, "an array is not aligned to its elements%s%s");
  return EBR_OK;
}

size_t round16(size_t b) { return (b + 15) & ~size_t{15}; }

// Run fn(tag of A, tag of B) for two I/O types.
template <typename Fn>
int with_types(int a, int b, Fn&& fn) {
  return with_type(a, [&](auto* ta) -> int {
    if constexpr (std::is_same_v<std::remove_pointer_t<decltype(ta)>, double>) {
      return set_error(EBR_ERR_DTYPE, "float64 is not a type of this operator%s%s");
    } else {
      return with_type(b, [&](auto* tb) -> int {
        if constexpr (std::is_same_v<std::remove_pointer_t<decltype(tb)>, double>)
          return set_error(EBR_ERR_DTYPE, "float64 is not a type of this operator%s%s");
        else
          return fn(ta, tb);
      });
    }
  });
}

// Run fn(integral constant V) with the widest V of {8, 4, 2, 1} (at most `most`) for which rows of C elements and the
// given row strides and pointers keep every access of V elements of `size` bytes (16 at most) aligned.
struct Rows {
  const void* p;
  int64_t stride;
  int size;
};

int access_width(int most, int64_t C, std::initializer_list<Rows> rows) {
  int v = most;
  for (; v > 1; v /= 2) {
    bool ok = C % v == 0;
    for (const Rows& r : rows) {
      const int64_t bytes = std::min<int64_t>(16, static_cast<int64_t>(v) * r.size);
      ok = ok && reinterpret_cast<uintptr_t>(r.p) % bytes == 0 && (r.stride * r.size) % bytes == 0;
    }
    if (ok) break;
  }
  return v;
}

// Vectors of a row that a warp of the expert kernels has in flight: two of the widest, eight of single elements.
constexpr int unroll_of(int v) { return v >= 8 ? 2 : v == 4 ? 4 : 8; }

template <int kMost, typename Fn>
int with_width(int v, Fn&& fn) {
  switch (v) {
    case 8:
      if constexpr (kMost >= 8) return fn(std::integral_constant<int, 8>{});
    case 4: return fn(std::integral_constant<int, 4>{});
    case 2: return fn(std::integral_constant<int, 2>{});
    default: return fn(std::integral_constant<int, 1>{});
  }
}

// ------------------------------------------------------------------------------------------------ sort

// Keys that one cluster of 16 CTAs ranks in registers, and those up to which it is used even where nothing runs
// beside it: 18,006 slots take 8.7 us in a cluster; 124,416 take 15.6 there and 7.0 in two kernels over the whole
// GPU.
constexpr int64_t kClusterKeys = 16 * int64_t{ebr::keysort::kSortThreads} * 16;
constexpr int64_t kClusterAlone = 32 * 1024;

// Bytes of zeros from which the sort in one cluster hides behind the zeroing, and up to which the sort's own blocks
// write them.
constexpr int64_t kHidingBytes = 64 << 20;
constexpr int64_t kSmallZeroBytes = 1 << 20;

bool sort_in_cluster(int64_t n, int64_t zero_bytes) {
  return n <= kClusterAlone || (n <= kClusterKeys && zero_bytes >= kHidingBytes);
}

int digit_passes(int64_t range) {  // keys in [0, range]
  int bits = 1;
  while ((int64_t{1} << bits) <= range) ++bits;
  return (bits + ebr::keysort::kMaxDigitBits - 1) / ebr::keysort::kMaxDigitBits;
}

int digit_bits(int64_t range, int passes) {
  int bits = 1;
  while ((int64_t{1} << bits) <= range) ++bits;
  return (bits + passes - 1) / passes;
}

// Items per thread and tiles of the whole-grid sort.
int sort_items(int64_t n) { return n <= int64_t{2} * ebr::keysort::kSortThreads * ebr::keysort::kMaxTiles ? 2 : 8; }
int64_t sort_tiles(int64_t n) {
  const int64_t tile = static_cast<int64_t>(sort_items(n)) * ebr::keysort::kSortThreads;
  return (n + tile - 1) / tile;
}

// Scratch of a sort: two (key, position) arrays where there is output, and the whole-grid path's counts.
size_t sort_scratch(int64_t n, int64_t digits, int passes, bool route) {
  size_t b = 0;
  if (!route) b += (passes > 1 ? 4 : 2) * round16(static_cast<size_t>(n) * 4);
  if (n > kClusterAlone) b += round16(static_cast<size_t>(digits) * sort_tiles(n) * 4) + round16(digits * 4);
  return b;
}

template <int kItems>
int launch_cluster_sort(int device, const ClusterSort& a, int ctas, int bits, cudaStream_t st) {
  auto* kernel = ebr::keysort::cluster_sort_kernel<kItems>;
  static std::atomic<bool> ready[kMaxDevices];
  if (device >= kMaxDevices || !ready[device].load()) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(ebr::keysort::cluster_sort_smem(ebr::keysort::kMaxDigitBits)));
    if (e != cudaSuccess) return cuda_error(e, "cluster sort attributes");
    if (device < kMaxDevices) ready[device].store(true);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(ebr::keysort::kSortThreads);
  cfg.dynamicSmemBytes = ebr::keysort::cluster_sort_smem(bits);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {static_cast<unsigned>(ctas), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) return cuda_error(e, "cluster sort");
  return check_launch("cluster sort");
}

// Zeros, beside the cluster sort that was launched before where `beside`.
int launch_zero(void* p, int64_t bytes, bool beside, cudaStream_t st) {
  if (bytes == 0) return EBR_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((bytes + ebr::keysort::kZeroPiece - 1) / ebr::keysort::kZeroPiece));
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = beside ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, ebr::keysort::zero_kernel, static_cast<char*>(p), bytes);
  if (e != cudaSuccess) return cuda_error(e, "zeroing");
  return check_launch("zeroing");
}

template <int kItems>
int launch_grid_sort(int device, GridSort& g, const ebr::keysort::Pass* pass, int passes, cudaStream_t st) {
  const size_t smem = ebr::keysort::grid_place_smem(g.digits);
  // The limit is the kernel's, not the call's: always the largest, so that no thread lowers it under another's launch.
  static std::atomic<bool> ready[kMaxDevices];
  if (device >= kMaxDevices || !ready[device].load()) {
    const cudaError_t e =
        cudaFuncSetAttribute(ebr::keysort::grid_place_kernel<kItems>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(ebr::keysort::grid_place_smem(1 << ebr::keysort::kMaxDigitBits)));
    if (e != cudaSuccess) return cuda_error(e, "sort attributes");
    if (device < kMaxDevices) ready[device].store(true);
  }
  g.scanned = g.tiles > ebr::keysort::kMaxTiles;
  for (int p = 0; p < passes; ++p) {
    g.pass = pass[p];
    ebr::keysort::grid_count_kernel<kItems><<<g.tiles, ebr::keysort::kSortThreads, 0, st>>>(g);
    int rc = check_launch("sort count");
    if (rc != EBR_OK) return rc;
    if (g.scanned) {
      ebr::keysort::grid_scan_kernel<<<g.digits, ebr::keysort::kSortThreads, 0, st>>>(g);
      if ((rc = check_launch("sort scan")) != EBR_OK) return rc;
    }
    ebr::keysort::grid_place_kernel<kItems><<<g.tiles, ebr::keysort::kSortThreads, smem, st>>>(g);
    if ((rc = check_launch("sort place")) != EBR_OK) return rc;
  }
  return EBR_OK;
}

// Sort n keys of [0, range]; digits: of one pass. For a route (route.row_of set) there is one pass, else the sorted
// keys and positions are at *key / *order in the scratch. `zero_bytes` at `zero` (16-byte aligned) are zeroed beside
// or before the sort.
int run_sort(int device, IdSource src, int64_t n, int passes, int bits, const ebr::keysort::RouteOut& route,
             void* scratch, int** key, int** order, void* zero, int64_t zero_bytes, cudaStream_t st) {
  char* at = static_cast<char*>(scratch);
  auto take = [&](size_t bytes) {
    char* p = at;
    at += round16(bytes);
    return reinterpret_cast<int*>(p);
  };
  ebr::keysort::Pass pass[3] = {};
  const bool is_route = route.row_of != nullptr;
  if (!is_route) {
    int* buf[4] = {take(n * 4), take(n * 4), nullptr, nullptr};
    if (passes > 1) {
      buf[2] = take(n * 4);
      buf[3] = take(n * 4);
    }
    for (int p = 0; p < passes; ++p) {
      const int to = (passes - 1 - p) % 2;  // the last pass writes the first pair
      pass[p].key_in = p ? buf[2 * (1 - to)] : nullptr;
      pass[p].idx_in = p ? buf[2 * (1 - to) + 1] : nullptr;
      pass[p].key_out = buf[2 * to];
      pass[p].idx_out = buf[2 * to + 1];
      pass[p].shift = p * bits;
      pass[p].bits = bits;
    }
    *key = buf[0];
    *order = buf[1];
  } else {
    pass[0].bits = bits;
  }
  ebr::keysort::SmallZero small = {nullptr, 0};
  if (zero_bytes <= kSmallZeroBytes) {
    small = {static_cast<char*>(zero), zero_bytes};
    zero_bytes = 0;
  }
  if (sort_in_cluster(n, zero_bytes)) {
    ClusterSort a = {};
    a.zero = small;
    a.src = src;
    a.n = n;
    a.passes = passes;
    for (int p = 0; p < 3; ++p) a.pass[p] = pass[p];
    a.route = route;
    int ctas = 1;
    while (ctas < 16 && static_cast<int64_t>(ctas) * ebr::keysort::kSortThreads < n) ctas *= 2;
    const int64_t per_thread = ((n + ctas - 1) / ctas + ebr::keysort::kSortThreads - 1) / ebr::keysort::kSortThreads;
    const int rc = per_thread <= 1   ? launch_cluster_sort<1>(device, a, ctas, bits, st)
                   : per_thread <= 2 ? launch_cluster_sort<2>(device, a, ctas, bits, st)
                   : per_thread <= 4 ? launch_cluster_sort<4>(device, a, ctas, bits, st)
                   : per_thread <= 8 ? launch_cluster_sort<8>(device, a, ctas, bits, st)
                                     : launch_cluster_sort<16>(device, a, ctas, bits, st);
    return rc != EBR_OK ? rc : launch_zero(zero, zero_bytes, true, st);
  }
  const int rc = launch_zero(zero, zero_bytes, false, st);
  if (rc != EBR_OK) return rc;
  GridSort g = {};
  g.zero = small;
  g.src = src;
  g.n = n;
  g.digits = is_route ? route.experts : 1 << bits;
  g.tiles = static_cast<int>(sort_tiles(n));
  g.counts = take(static_cast<size_t>(g.digits) * g.tiles * 4);
  g.totals = take(static_cast<size_t>(g.digits) * 4);
  g.route = route;
  return sort_items(n) == 2 ? launch_grid_sort<2>(device, g, pass, passes, st)
                            : launch_grid_sort<8>(device, g, pass, passes, st);
}

// ------------------------------------------------------------------------------------------------ embedding

int check_embedding(int id_type, int64_t n, int64_t V, int64_t C, int64_t stride) {
  int rc = check_id_type(id_type);
  if (rc != EBR_OK) return rc;
  if (n < 0 || V < 1 || C < 1) return set_error(EBR_ERR_SHAPE, "embedding: bad sizes%s%s");
  if (n >= kMaxSortKeys || V >= kMaxSortKeys || C > (1 << 24))
    return set_error(EBR_ERR_SHAPE, "embedding: size too large%s%s");
  if (stride < 0) return set_error(EBR_ERR_STRIDE, "embedding: negative stride%s%s");
  return EBR_OK;
}

// Rows of a chunk of the gradient, 8 to 256: up to 3,500 warps' worth of chunks. 62,208 board tokens of 512 columns:
// the whole gradient takes 26.6 us warm and 39 cold with 64 rows, 32.8 and 47 with 32, which leave twice the partial
// sums to join, 28.7 and 45 with 128, which leave half the warps.
int64_t grad_chunk_rows(int64_t n, int64_t C) {
  const int64_t blocks = (C + 255) / 256;
  int64_t r = 8;
  while (r < 256 && n * blocks / r > 3500) r *= 2;
  return r;
}

// Gradients that one launch makes, the warps looking through all ids: few tokens, and as many warps as some waves of
// them. A block owns a table row where the rows are few, up to kSomeTokens (500 tokens over ten ids: 4.2 us, 12.7 by
// way of the sort), else a warp does, up to kFewTokens.
constexpr int64_t kFewTokens = 128, kSomeTokens = 512;

bool grad_by_blocks(int64_t n, int64_t V, int64_t C) { return n <= kSomeTokens && V * ((C + 255) / 256) <= 2048; }
bool grad_by_few(int64_t n, int64_t V, int64_t C) {
  return grad_by_blocks(n, V, C) || (n <= kFewTokens && V * ((C + 255) / 256) <= 65536);
}

// ------------------------------------------------------------------------------------------------ distillation

constexpr int64_t kMaxVocabulary = int64_t{1} << 19;
constexpr int kMaxEntries = 1024;
// The long rows' kernel counts rows in an int, in steps of up to six clusters for each SM: the last step has to fit, too.
constexpr int64_t kMaxRows = (int64_t{1} << 31) - (1 << 16);
constexpr double kLeastTau = 0x1p-126;  // the smallest normal float: log2(e) / tau is finite

// Rows of a few logits take four lanes each, rows of up to kWarpRowBytes a warp (half as much where there are not
// rows enough to fill the GPU so), longer ones a ring of chunks. bfloat16, 2.1 GB of logits and gradient: a warp
// takes 0.52 ms at V = 8,192 (the ring 0.72) and 0.57 at 16,384 (0.60).
constexpr int64_t kWarpRowBytes = 32 * 1024;

bool distill_few(int64_t V, int64_t K) { return V <= 32 && K <= 32; }

template <typename T, bool kStats>
int launch_distill_few(const ebr::distill::Args& a, cudaStream_t st) {
  using namespace ebr::distill;
  constexpr int kLanes = 4, kGroups = kSmallThreads / kLanes;
  distill_small_kernel<T, kLanes, kStats><<<static_cast<unsigned>((a.N + kGroups - 1) / kGroups), kSmallThreads,
                                            static_cast<size_t>(kGroups) * 2 * a.K * 4, st>>>(a);
  return check_launch("topk_distill");
}

template <typename T>
bool distill_by_warp(int64_t N, int64_t V) {
  return V * static_cast<int64_t>(sizeof(T)) <= (N >= 256 ? kWarpRowBytes : kWarpRowBytes / 2);
}

template <typename T, bool kStats>
int launch_distill_warp(const ebr::distill::Args& a, cudaStream_t st) {
  using namespace ebr::distill;
  distill_warp_kernel<T, kStats><<<static_cast<unsigned>((a.N + kMidWarps - 1) / kMidWarps), kMidWarps * 32,
                                   static_cast<size_t>(kMidWarps) * 12 * a.K, st>>>(a);
  return check_launch("topk_distill");
}

template <typename T, int kWarps, int kU>
int launch_distill_row(int device, const ebr::distill::Args& a, int slices, int granules, int slots, int per_sm,
                       cudaStream_t st) {
  auto* kernel = ebr::distill::distill_row_kernel<T, kWarps, kU>;
  static std::atomic<bool> ready[kMaxDevices];
  if (device >= kMaxDevices || !ready[device].load()) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 216 * 1024);
    if (e != cudaSuccess) return cuda_error(e, "topk_distill attributes");
    if (device < kMaxDevices) ready[device].store(true);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kWarps * 32 + 32);
  cfg.dynamicSmemBytes = static_cast<size_t>(slots) * kWarps * kU * 512;
  const int64_t clusters = std::max<int64_t>(1, std::min<int64_t>(a.N, per_sm * sm_count(device) / slices));
  // The rows' weights come from a kernel of their own (in `losses`, which the last kernel writes), unless no cluster
  // has a second row: 12 rows of 151,665 float16 logits take 8.2 us without it, 9.5 with it.
  const float* weights = clusters < a.N ? a.losses : nullptr;
  if (weights) {
    ebr::distill::distill_weights_kernel<<<static_cast<unsigned>((a.N + 7) / 8), 256, 0, st>>>(a, a.losses);
    const int rc = check_launch("topk_distill weights");
    if (rc != EBR_OK) return rc;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * slices));
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {static_cast<unsigned>(slices), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, weights, slices, granules, slots);
  if (e != cudaSuccess) return cuda_error(e, "topk_distill");
  return check_launch("topk_distill");
}

template <typename T, bool kLoss>
int launch_distill_entries(const ebr::distill::Args& a, cudaStream_t st) {
  using namespace ebr::distill;
  distill_entries_kernel<T, kLoss><<<static_cast<unsigned>((a.N + kEntryWarps - 1) / kEntryWarps), kEntryWarps * 32,
                                     static_cast<size_t>(kEntryWarps) * 3 * a.K * 4, st>>>(a);
  return check_launch("topk_distill entries");
}

// 16-byte granules that a row of V elements may touch, whatever its first byte.
template <typename T>
int64_t row_granules(int64_t V) {
  constexpr int64_t kE = 16 / sizeof(T);
  return (V + 2 * (kE - 1)) / kE;
}

template <typename T>
int launch_distill(int device, const ebr::distill::Args& a, cudaStream_t st) {
  if (distill_few(a.V, a.K)) return launch_distill_few<T, true>(a, st);
  if (distill_by_warp<T>(a.N, a.V)) return launch_distill_warp<T, true>(a, st);
  const int64_t total = row_granules<T>(a.V);
  int slices = 1;
  while (slices < ebr::distill::kMaxSlices && a.N * slices < 2 * sm_count(device) && (total + slices - 1) / slices > 256)
    slices *= 2;
  const int granules = static_cast<int>((total + slices - 1) / slices);
  // Slices above 128 KB (a row's, where it is not split): rings of four 24 KB chunks, two on an SM, 24 warps; shorter
  // ones want more rows in flight: rings of four 8 KB chunks, six on an SM. bfloat16 at 2.1 GB: V = 131,072 takes
  // 0.44 ms with the first, 0.55 with the second; V = 32,768 takes 0.56 and 0.50.
  const int rc = granules > 8192 ? launch_distill_row<T, 12, 4>(device, a, slices, granules, 4, 2, st)
                                 : launch_distill_row<T, 4, 4>(device, a, slices, granules, 4, 6, st);
  return rc != EBR_OK ? rc : launch_distill_entries<T, true>(a, st);
}

template <typename T>
int launch_distill_grad(int device, const ebr::distill::Args& a, cudaStream_t st) {
  if (distill_few(a.V, a.K)) return launch_distill_few<T, false>(a, st);
  if (distill_by_warp<T>(a.N, a.V)) return launch_distill_warp<T, false>(a, st);
  constexpr int kThreads = 256;
  const int64_t total = row_granules<T>(a.V);
  if (a.unless_one) {
    ebr::distill::distill_grad_kernel<T, kThreads, true>
        <<<static_cast<unsigned>(std::min<int64_t>(a.N, static_cast<int64_t>(sm_count(device)) * 4)), kThreads,
           static_cast<size_t>(a.K) * 12, st>>>(a, 1, static_cast<int>(total));
    return check_launch("topk_distill_grad");
  }
  const int slices = static_cast<int>((total + 4095) / 4096);
  const int64_t blocks = std::min(a.N * slices, static_cast<int64_t>(sm_count(device)) * 64);
  ebr::distill::distill_grad_kernel<T, kThreads, false><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(
      a, slices, static_cast<int>((total + slices - 1) / slices));
  const int rc = check_launch("topk_distill_grad");
  return rc != EBR_OK ? rc : launch_distill_entries<T, false>(a, st);
}

int check_distill(int dtype, int id_type, int top_dtype, int64_t N, int64_t V, int64_t K, double tau, int64_t stride,
                  int64_t grad_stride) {
  int rc = check_layer_dtype(dtype, false);
  if (rc == EBR_OK) rc = check_layer_dtype(top_dtype, false);
  if (rc == EBR_OK) rc = check_id_type(id_type);
  if (rc != EBR_OK) return rc;
  if (N < 0 || V < 1 || K < 1 || K > kMaxEntries) return set_error(EBR_ERR_SHAPE, "topk_distill: bad sizes%s%s");
  if (N >= kMaxRows || V > kMaxVocabulary) return set_error(EBR_ERR_SHAPE, "topk_distill: size too large%s%s");
  if (!(tau >= kLeastTau && tau <= 1e30))
    return set_error(EBR_ERR_SHAPE, "topk_distill: the temperature must be between 1.2e-38 and 1e30%s%s");
  if (stride < 0 || grad_stride < V) return set_error(EBR_ERR_STRIDE, "topk_distill: bad row stride%s%s");
  return EBR_OK;
}

ebr::distill::Args distill_args(int64_t N, int64_t V, int64_t K, double tau, double factor, int id_type, int top_dtype,
                                const void* logits, int64_t stride, const void* ids, const void* top,
                                const float* row_weight) {
  ebr::distill::Args a = {};
  a.N = N;
  a.V = V;
  a.K = static_cast<int>(K);
  a.tau = static_cast<float>(tau);
  a.exp2_scale = static_cast<float>(1.4426950408889634 / tau);
  a.factor = static_cast<float>(factor);
  a.logits = logits;
  a.logits_stride = stride;
  a.top_ids = ids;
  a.ids64 = id_type == EBR_INT64;
  a.top_logits = top;
  a.top_dtype = top_dtype;
  a.row_weight = row_weight;
  return a;
}

}  // namespace

extern "C" {

int ebr_scaled_embedding(int w_dtype, int out_dtype, int id_type, int64_t n, int64_t V, int64_t C, double scale,
                         const void* ids, const void* w, int64_t w_stride, void* out, void* stream) {
  int rc = check_embedding(id_type, n, V, C, w_stride);
  if (rc == EBR_OK) rc = check_layer_dtype(w_dtype, false);
  if (rc == EBR_OK) rc = check_layer_dtype(out_dtype, false);
  if (rc != EBR_OK) return rc;
  if (n == 0) return EBR_OK;
  if (!ids || !w || !out) return set_error(EBR_ERR_NULL, "scaled_embedding: NULL pointer%s%s");
  if ((rc = check_ids(ids, id_type)) != EBR_OK) return rc;
  if ((rc = check_arrays({{w, elem_size(w_dtype)}, {out, elem_size(out_dtype)}})) != EBR_OK) return rc;
  int device = 0;
  if ((rc = check_device(&device)) != EBR_OK) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  return with_types(w_dtype, out_dtype, [&](auto* wt, auto* ot) -> int {
    using TW = std::remove_pointer_t<decltype(wt)>;
    using TO = std::remove_pointer_t<decltype(ot)>;
    constexpr int kMost = sizeof(TW) == 4 && sizeof(TO) == 4 ? 4 : 8;
    const int v = access_width(kMost, C, {{w, w_stride, int(sizeof(TW))}, {out, C, int(sizeof(TO))}});
    return with_width<kMost>(v, [&](auto vc) -> int {
      constexpr int V_ = decltype(vc)::value;
      using namespace ebr::embed;
      constexpr int kU = V_ >= 4 ? 1 : 4;  // vectors of a row in flight: narrow ones need more
      const int64_t cols = (C + kU * 32 * V_ - 1) / (kU * 32 * V_);
      if (cols > 65535) return set_error(EBR_ERR_SHAPE, "scaled_embedding: row too long%s%s");
      // as many tokens to a warp (up to 32) as leave some 24 warps for each SM
      int per_warp = 1;
      while (per_warp < 32 && n * cols / per_warp > 24 * static_cast<int64_t>(sm_count(device))) per_warp *= 2;
      const int64_t blocks = (n + per_warp * kLookupWarps - 1) / (per_warp * kLookupWarps);
      lookup_kernel<TW, TO, V_, kU><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(cols)), kLookupWarps * 32,
                                  0, st>>>(IdSource{ids, id_type == EBR_INT64, static_cast<int>(V)}, n, C,
                                           static_cast<float>(scale), static_cast<const TW*>(w), w_stride,
                                           static_cast<TO*>(out), per_warp);
      return check_launch("scaled_embedding");
    });
  });
}

size_t ebr_scaled_embedding_grad_scratch_bytes(int64_t n, int64_t V, int64_t C) {
  if (n <= 0 || V < 1 || C < 1 || n >= kMaxSortKeys || V >= kMaxSortKeys || C > (1 << 24)) return 0;
  if (grad_by_few(n, V, C)) return 0;
  const int passes = digit_passes(V);
  const int64_t chunks = (n + grad_chunk_rows(n, C) - 1) / grad_chunk_rows(n, C);
  return sort_scratch(n, int64_t{1} << digit_bits(V, passes), passes, false) +
         round16(static_cast<size_t>(chunks) * 2 * C * 4);
}

int ebr_scaled_embedding_grad(int g_dtype, int w_dtype, int id_type, int64_t n, int64_t V, int64_t C, double scale,
                              const void* ids, const void* g, int64_t g_stride, void* dw, void* scratch,
                              size_t scratch_bytes, void* stream) {
  int rc = check_embedding(id_type, n, V, C, g_stride);
  if (rc == EBR_OK) rc = check_layer_dtype(g_dtype, false);
  if (rc == EBR_OK) rc = check_layer_dtype(w_dtype, false);
  if (rc != EBR_OK) return rc;
  if (!dw) return set_error(EBR_ERR_NULL, "scaled_embedding_grad: NULL pointer%s%s");
  const int64_t dw_bytes = V * C * static_cast<int64_t>(elem_size(w_dtype));
  auto st = static_cast<cudaStream_t>(stream);
  int device = 0;
  if (n == 0) {
    if ((rc = check_device(&device)) != EBR_OK) return rc;
    const cudaError_t e = cudaMemsetAsync(dw, 0, static_cast<size_t>(dw_bytes), st);
    return e == cudaSuccess ? EBR_OK : cuda_error(e, "scaled_embedding_grad");
  }
  if (!ids || !g) return set_error(EBR_ERR_NULL, "scaled_embedding_grad: NULL pointer%s%s");
  if ((rc = check_ids(ids, id_type)) != EBR_OK) return rc;
  if ((rc = check_arrays({{g, elem_size(g_dtype)}})) != EBR_OK) return rc;
  if (!aligned16(dw)) return set_error(EBR_ERR_STRIDE, "scaled_embedding_grad: dW must be 16-byte aligned%s%s");
  const size_t need = ebr_scaled_embedding_grad_scratch_bytes(n, V, C);
  if (need && (!scratch || !aligned16(scratch) || scratch_bytes < need))
    return set_error(EBR_ERR_SCRATCH, "scaled_embedding_grad: scratch too small or unaligned%s%s");
  if ((rc = check_device(&device)) != EBR_OK) return rc;
  if (!need)
    return with_types(g_dtype, w_dtype, [&](auto* gt, auto* wt) -> int {
      using TG = std::remove_pointer_t<decltype(gt)>;
      using TW = std::remove_pointer_t<decltype(wt)>;
      using namespace ebr::embed;
      constexpr int kMost = static_cast<int>(16 / sizeof(TG));
      const int v = access_width(kMost, C, {{g, g_stride, int(sizeof(TG))}, {dw, C, int(sizeof(TW))}});
      return with_width<kMost>(v, [&](auto vc) -> int {
        constexpr int V_ = decltype(vc)::value;
        const int64_t cols = (C + 32 * V_ - 1) / (32 * V_);
        if (cols > 65535) return set_error(EBR_ERR_SHAPE, "scaled_embedding_grad: row too long%s%s");
        const IdSource src{ids, id_type == EBR_INT64, static_cast<int>(V)};
        auto launch = [&](auto share) {
          constexpr int kShare = decltype(share)::value, kOwners = kGradWarps / kShare;
          grad_few_kernel<TG, TW, V_, kShare><<<dim3(static_cast<unsigned>((V + kOwners - 1) / kOwners),
                                                     static_cast<unsigned>(cols)), kGradWarps * 32, 0, st>>>(
              src, static_cast<int>(n), C, static_cast<const TG*>(g), g_stride, static_cast<float>(scale),
              static_cast<TW*>(dw));
        };
        if (grad_by_blocks(n, V, C))
          launch(std::integral_constant<int, kGradWarps>{});
        else
          launch(std::integral_constant<int, 1>{});
        return check_launch("scaled_embedding_grad");
      });
    });
  const int passes = digit_passes(V), bits = digit_bits(V, passes);
  int *key = nullptr, *order = nullptr;
  const IdSource src{ids, id_type == EBR_INT64, static_cast<int>(V)};
  rc = run_sort(device, src, n, passes, bits, {}, scratch, &key, &order, dw, dw_bytes, st);
  if (rc != EBR_OK) return rc;
  float* part = reinterpret_cast<float*>(static_cast<char*>(scratch) +
                                         sort_scratch(n, int64_t{1} << bits, passes, false));
  const int R = static_cast<int>(grad_chunk_rows(n, C));
  const int64_t chunks = (n + R - 1) / R;
  return with_types(g_dtype, w_dtype, [&](auto* gt, auto* wt) -> int {
    using TG = std::remove_pointer_t<decltype(gt)>;
    using TW = std::remove_pointer_t<decltype(wt)>;
    using namespace ebr::embed;
    constexpr int kMost = static_cast<int>(16 / sizeof(TG));
    const int v = access_width(kMost, C, {{g, g_stride, int(sizeof(TG))}, {dw, C, int(sizeof(TW))}, {part, C, 4}});
    int r = with_width<kMost>(v, [&](auto vc) -> int {
      constexpr int V_ = decltype(vc)::value;
      const int64_t cols = (C + 32 * V_ - 1) / (32 * V_);
      if (cols > 65535) return set_error(EBR_ERR_SHAPE, "scaled_embedding_grad: row too long%s%s");
      grad_chunk_kernel<TG, TW, V_><<<dim3(static_cast<unsigned>((chunks + kGradWarps - 1) / kGradWarps),
                                           static_cast<unsigned>(cols)), kGradWarps * 32, 0, st>>>(
          static_cast<int>(n), static_cast<int>(V), C, R, key, order, static_cast<const TG*>(g), g_stride,
          static_cast<float>(scale), static_cast<TW*>(dw), part);
      return check_launch("scaled_embedding_grad");
    });
    if (r != EBR_OK || chunks == 1) return r;
    const int64_t cols = (C + 127) / 128;
    if (cols > 65535) return set_error(EBR_ERR_SHAPE, "scaled_embedding_grad: row too long%s%s");
    grad_join_kernel<TW><<<dim3(static_cast<unsigned>((chunks + kJoinChunks - 1) / kJoinChunks),
                                static_cast<unsigned>(cols)), kJoinWarps * 32, 0, st>>>(
        static_cast<int>(n), static_cast<int>(V), C, R, static_cast<int>(chunks), key, static_cast<float>(scale),
        static_cast<TW*>(dw), part);
    return check_launch("scaled_embedding_grad join");
  });
}

}  // extern "C"

namespace {
// Blocks along the tokens, each warp walking over several of them where there are many (board batch: dispatch 42 us
// with a warp for each token, 38 so), and along the columns, where the tokens alone leave less than 96 warps to an SM
// (3,001 tokens of 999 float32, six rows each: cold, combine 54 us without, 29 with).
dim3 expert_grid(int device, int64_t T, int64_t C, int per_trip, bool split) {
  const int64_t warps = int64_t{96} * sm_count(device);
  const int64_t parts = split ? std::max<int64_t>(1, std::min((C + per_trip - 1) / per_trip, warps / std::max<int64_t>(T, 1))) : 1;
  const int64_t blocks = std::min<int64_t>((T + ebr::experts::kWarps - 1) / ebr::experts::kWarps, 24 * int64_t{sm_count(device)});
  return dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(std::min<int64_t>(parts, 64)));
}
}  // namespace

extern "C" {

size_t ebr_expert_route_scratch_bytes(int64_t T, int64_t K, int64_t E) {
  if (T <= 0 || K <= 0 || E < 1 || E > kMaxExperts || T >= kMaxSortKeys || K >= kMaxSortKeys || T * K >= kMaxSortKeys)
    return 0;
  return sort_scratch(T * K, E, 1, true);
}

int ebr_expert_route(int id_type, int64_t T, int64_t K, int64_t E, int64_t capacity, const void* ids, int32_t* row_of,
                     int32_t* slot_of, int32_t* offsets, void* scratch, size_t scratch_bytes, void* stream) {
  int rc = check_id_type(id_type);
  if (rc != EBR_OK) return rc;
  if (T < 0 || K < 1 || E < 1 || E > kMaxExperts || capacity < 0) return set_error(EBR_ERR_SHAPE, "expert_route: bad sizes%s%s");
  if (T >= kMaxSortKeys || K >= kMaxSortKeys || T * K >= kMaxSortKeys || capacity >= kMaxSortKeys ||
      E * capacity >= kMaxSortKeys)
    return set_error(EBR_ERR_SHAPE, "expert_route: size too large%s%s");
  const int64_t n = T * K, rows = capacity ? E * capacity : n;
  if (!offsets || (n && (!ids || !row_of)) || (rows && !slot_of)) return set_error(EBR_ERR_NULL, "expert_route: NULL pointer%s%s");
  if ((rc = check_ids(ids, id_type)) != EBR_OK) return rc;
  if ((rc = check_arrays({{row_of, 4}, {slot_of, 4}, {offsets, 4}})) != EBR_OK) return rc;
  const size_t need = ebr_expert_route_scratch_bytes(T, K, E);
  if (need && (!scratch || !aligned16(scratch) || scratch_bytes < need))
    return set_error(EBR_ERR_SCRATCH, "expert_route: scratch too small or unaligned%s%s");
  int device = 0;
  if ((rc = check_device(&device)) != EBR_OK) return rc;
  int bits = 0;
  while ((1 << bits) < E) ++bits;
  ebr::keysort::RouteOut route = {};
  route.row_of = row_of ? row_of : offsets;  // no slot: only marks the sort as a route
  route.slot_of = slot_of;
  route.offsets = offsets;
  route.experts = static_cast<int>(E);
  route.capacity = capacity;
  route.rows = rows;
  return run_sort(device, IdSource{ids, id_type == EBR_INT64, static_cast<int>(E)}, n, 1, bits, route, scratch, nullptr,
                  nullptr, nullptr, 0, static_cast<cudaStream_t>(stream));
}

int ebr_expert_scatter(int dtype, int weight_dtype, int64_t T, int64_t K, int64_t C, int64_t rows, const void* x,
                       int64_t x_stride, const int32_t* row_of, const int32_t* slot_of, const void* weights,
                       const void* rows_in, void* rows_out, void* dots, void* stream) {
  int rc = check_layer_dtype(dtype, false);
  if (rc != EBR_OK) return rc;
  if (weight_dtype != EBR_FLOAT32 && weight_dtype != dtype)
    return set_error(EBR_ERR_DTYPE, "expert_scatter: weights must be float32 or of the rows' type%s%s");
  if (T < 0 || K < 1 || C < 1 || rows < 0 || T >= kMaxSortKeys || K >= kMaxSortKeys || T * K >= kMaxSortKeys ||
      rows >= kMaxSortKeys || C > (1 << 24))
    return set_error(EBR_ERR_SHAPE, "expert_scatter: bad sizes%s%s");
  if (x_stride < 0) return set_error(EBR_ERR_STRIDE, "expert_scatter: negative stride%s%s");
  if (!rows_out && !dots) return set_error(EBR_ERR_NULL, "expert_scatter: no output%s%s");
  if ((rows_in == nullptr) != (dots == nullptr) && T * rows != 0)
    return set_error(EBR_ERR_NULL, "expert_scatter: rows_in and dots go together%s%s");
  if ((T && (!x || !row_of)) || (rows && rows_out && !slot_of)) return set_error(EBR_ERR_NULL, "expert_scatter: NULL pointer%s%s");
  if (T == 0 && (rows == 0 || !rows_out)) return EBR_OK;
  const size_t size_x = elem_size(dtype), size_w = elem_size(weight_dtype);
  rc = check_arrays({{x, size_x}, {rows_in, size_x}, {rows_out, size_x}, {row_of, 4}, {slot_of, 4}, {weights, size_w},
                     {dots, size_w}});
  if (rc != EBR_OK) return rc;
  int device = 0;
  if ((rc = check_device(&device)) != EBR_OK) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  return with_type(dtype, [&](auto* tag) -> int {
    using T_ = std::remove_pointer_t<decltype(tag)>;
    if constexpr (std::is_same_v<T_, double>) {
      return EBR_ERR_DTYPE;
    } else {
      constexpr int size = sizeof(T_), kMost = 16 / size;
      const int v = access_width(kMost, C, {{x, x_stride, size}, {rows_in, C, size}, {rows_out, C, size}});
      return with_width<kMost>(v, [&](auto vc) -> int {
        constexpr int V_ = decltype(vc)::value;
        auto launch = [&](auto* wtag, auto with_dots) -> int {
          using TW = std::remove_pointer_t<decltype(wtag)>;
          using namespace ebr::experts;
          const dim3 grid = expert_grid(device, T, C, unroll_of(V_) * 32 * V_, dots == nullptr);
          const int64_t tb = grid.x;
          const int64_t zb = rows_out ? (rows + kZeroRows - 1) / kZeroRows : 0;
          scatter_kernel<T_, TW, V_, unroll_of(V_), decltype(with_dots)::value><<<dim3(static_cast<unsigned>(tb + zb), grid.y), kWarps * 32, 0, st>>>(
              T, static_cast<int>(K), C, rows, static_cast<const T_*>(x), x_stride, row_of, slot_of,
              static_cast<const TW*>(weights), static_cast<const T_*>(rows_in), static_cast<T_*>(rows_out),
              static_cast<TW*>(dots), static_cast<int>(tb));
          return check_launch("expert_scatter");
        };
        if (weight_dtype == EBR_FLOAT32)
          return dots ? launch(static_cast<float*>(nullptr), std::true_type{})
                      : launch(static_cast<float*>(nullptr), std::false_type{});
        return dots ? launch(static_cast<T_*>(nullptr), std::true_type{})
                    : launch(static_cast<T_*>(nullptr), std::false_type{});
      });
    }
  });
}

int ebr_expert_combine(int dtype, int weight_dtype, int64_t T, int64_t K, int64_t C, const void* rows_in,
                       int64_t rows_stride, const int32_t* row_of, const void* weights, void* y, void* stream) {
  int rc = check_layer_dtype(dtype, false);
  if (rc != EBR_OK) return rc;
  if (weight_dtype != EBR_FLOAT32 && weight_dtype != dtype)
    return set_error(EBR_ERR_DTYPE, "expert_combine: weights must be float32 or of the rows' type%s%s");
  if (T < 0 || K < 1 || C < 1 || T >= kMaxSortKeys || K >= kMaxSortKeys || T * K >= kMaxSortKeys || C > (1 << 24))
    return set_error(EBR_ERR_SHAPE, "expert_combine: bad sizes%s%s");
  if (rows_stride < 0) return set_error(EBR_ERR_STRIDE, "expert_combine: negative stride%s%s");
  if (T == 0) return EBR_OK;
  if (!rows_in || !row_of || !y) return set_error(EBR_ERR_NULL, "expert_combine: NULL pointer%s%s");
  const size_t size_x = elem_size(dtype);
  if ((rc = check_arrays({{rows_in, size_x}, {y, size_x}, {row_of, 4}, {weights, elem_size(weight_dtype)}})) != EBR_OK)
    return rc;
  int device = 0;
  if ((rc = check_device(&device)) != EBR_OK) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  return with_type(dtype, [&](auto* tag) -> int {
    using T_ = std::remove_pointer_t<decltype(tag)>;
    if constexpr (std::is_same_v<T_, double>) {
      return EBR_ERR_DTYPE;
    } else {
      constexpr int size = sizeof(T_), kMost = 16 / size;
      const int v = access_width(kMost, C, {{rows_in, rows_stride, size}, {y, C, size}});
      return with_width<kMost>(v, [&](auto vc) -> int {
        constexpr int V_ = decltype(vc)::value;
        auto launch = [&](auto* wtag) -> int {
          using TW = std::remove_pointer_t<decltype(wtag)>;
          using namespace ebr::experts;
          combine_kernel<T_, TW, V_, unroll_of(V_)><<<expert_grid(device, T, C, unroll_of(V_) * 32 * V_, true), kWarps * 32, 0, st>>>(
              T, static_cast<int>(K), C, static_cast<const T_*>(rows_in), rows_stride, row_of,
              static_cast<const TW*>(weights), static_cast<T_*>(y));
          return check_launch("expert_combine");
        };
        return weight_dtype == EBR_FLOAT32 ? launch(static_cast<float*>(nullptr)) : launch(static_cast<T_*>(nullptr));
      });
    }
  });
}

int ebr_topk_distill(int dtype, int id_type, int top_dtype, int64_t N, int64_t V, int64_t K, double tau, double factor,
                     const void* logits, int64_t logits_stride, const void* top_ids, const void* top_logits,
                     const float* row_weight, float* losses, float* stats, float* total, void* grad, int64_t grad_stride,
                     void* stream) {
  int rc = check_distill(dtype, id_type, top_dtype, N, V, K, tau, logits_stride, grad ? grad_stride : V);
  if (rc != EBR_OK) return rc;
  if (N == 0 && !total) return EBR_OK;
  if (N && (!logits || !top_ids || !top_logits || !losses || !stats)) return set_error(EBR_ERR_NULL, "topk_distill: NULL pointer%s%s");
  if ((rc = check_ids(top_ids, id_type)) != EBR_OK) return rc;
  if (!on_boundary(stats, 8)) return set_error(EBR_ERR_STRIDE, "topk_distill: unaligned stats%s%s");
  rc = check_arrays({{logits, elem_size(dtype)}, {top_logits, elem_size(top_dtype)}, {row_weight, 4}, {losses, 4},
                     {total, 4}, {grad, elem_size(dtype)}});
  if (rc != EBR_OK) return rc;
  int device = 0;
  if ((rc = check_device(&device)) != EBR_OK) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  if (N) {
    ebr::distill::Args a = distill_args(N, V, K, tau, factor, id_type, top_dtype, logits, logits_stride, top_ids,
                                        top_logits, row_weight);
    a.losses = losses;
    a.stats = stats;
    a.grad = grad;
    a.grad_stride = grad_stride;
    rc = with_type(dtype, [&](auto* tag) -> int {
      using T = std::remove_pointer_t<decltype(tag)>;
      if constexpr (std::is_same_v<T, double>) return EBR_ERR_DTYPE;
      else return launch_distill<T>(device, a, st);
    });
    if (rc != EBR_OK) return rc;
  }
  if (!total) return EBR_OK;
  ebr::distill::total_kernel<<<1, 1024, 0, st>>>(N, static_cast<float>(factor), losses, total);
  return check_launch("topk_distill total");
}

int ebr_topk_distill_grad(int dtype, int id_type, int top_dtype, int64_t N, int64_t V, int64_t K, double tau,
                          double factor, const void* logits, int64_t logits_stride, const void* top_ids,
                          const void* top_logits, const float* row_weight, const float* stats, const float* upstream,
                          int64_t upstream_stride, int unless_one, void* grad, int64_t grad_stride, void* stream) {
  int rc = check_distill(dtype, id_type, top_dtype, N, V, K, tau, logits_stride, grad_stride);
  if (rc != EBR_OK) return rc;
  if (upstream_stride != 0 && upstream_stride != 1) return set_error(EBR_ERR_STRIDE, "topk_distill_grad: upstream stride must be 0 or 1%s%s");
  if (N == 0) return EBR_OK;
  if (!logits || !top_ids || !top_logits || !stats || !upstream || !grad)
    return set_error(EBR_ERR_NULL, "topk_distill_grad: NULL pointer%s%s");
  if ((rc = check_ids(top_ids, id_type)) != EBR_OK) return rc;
  if (!on_boundary(stats, 8)) return set_error(EBR_ERR_STRIDE, "topk_distill_grad: unaligned stats%s%s");
  rc = check_arrays({{logits, elem_size(dtype)}, {top_logits, elem_size(top_dtype)}, {row_weight, 4}, {upstream, 4},
                     {grad, elem_size(dtype)}});
  if (rc != EBR_OK) return rc;
  int device = 0;
  if ((rc = check_device(&device)) != EBR_OK) return rc;
  ebr::distill::Args a = distill_args(N, V, K, tau, factor, id_type, top_dtype, logits, logits_stride, top_ids,
                                      top_logits, row_weight);
  a.stats = const_cast<float*>(stats);
  a.upstream = upstream;
  a.upstream_stride = upstream_stride;
  a.unless_one = unless_one && upstream_stride == 0;
  a.grad = grad;
  a.grad_stride = grad_stride;
  return with_type(dtype, [&](auto* tag) -> int {
    using T = std::remove_pointer_t<decltype(tag)>;
    if constexpr (std::is_same_v<T, double>) return EBR_ERR_DTYPE;
    else return launch_distill_grad<T>(device, a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
