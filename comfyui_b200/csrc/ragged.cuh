// What the products over ragged groups of rows share: the rows of each group, the order of the tiles, tensor maps.
#pragma once
#include <cstring>
#include <type_traits>
#include <cuda.h>

#include "moe_common.cuh"
#include "ptx_sm100.cuh"

namespace comfy_b200 {

constexpr int kRaggedMaxGroups = COMFY_MOE_RAGGED_MAX_GROUPS;
constexpr int kRaggedThreads = 320;            // warp 0 = TMA producer, warp 1 = MMA issuer, warps 2-9 = epilogue,
constexpr int kRaggedTailThreads = 352;        // warp 10 = zeros behind a group (where the rows are the contraction)
constexpr int kRaggedEpilogueWarps = 8;        // two per TMEM lane quarter, each takes half of a tile's columns
constexpr int kStoreRowBytes = 64;             // one warp's store tile: 32 rows of 64 bytes, 64-byte swizzle
constexpr int kStoreTileBytes = 32 * kStoreRowBytes;

// Device-side status codes of a bounded wait that gave up.
constexpr int kStatusRaggedProducer = 10;
constexpr int kStatusRaggedMma = 11;
constexpr int kStatusRaggedEpilogue = 12;

// The rows of 32 groups, one to a lane of a whole warp, from what the caller left on the device:
//   begin[g] = max(offsets[0 .. g]) clipped to [0, rows],  end = the same up to g + 1,  count[g] = at most counts[g].
// Offsets that do not rise therefore give empty groups, never rows outside the buffers or rows that two groups share.
// `reach` carries the maximum from the 32 groups before these to the next ones; a lane behind the last group has no rows.
__device__ __forceinline__ void ragged_chunk(const int32_t* offsets, const int32_t* counts, int groups, int rows, int g,
                                             int& reach, int& begin, int& count) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = 0, most = 0;
  if (g < groups) {
    if (offsets) {
      lo = min(max(offsets[g], 0), rows);
      hi = min(max(offsets[g + 1], 0), rows);
    } else {
      hi = rows;                               // one group: all rows
    }
    most = counts ? max(counts[g], 0) : rows;
  }
  lo = max(lo, reach);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, max(lo, hi), d);
    if (lane >= d) lo = max(lo, v);
  }
  hi = max(lo, hi);
  begin = lo;
  count = min(hi - lo, most);
  reach = __shfl_sync(0xffffffffu, hi, 31);
}

// All groups' rows, made by one warp of every block.  first_tile[g] = tiles of the groups before g, for tiles of `tile_rows`
// rows (of one fixed number where tile_rows is 0).
__device__ __forceinline__ void ragged_ranges(const int32_t* offsets, const int32_t* counts, int groups, int rows,
                                              int tile_rows, int tiles_per_row_tile, int* begin, int* count,
                                              int* first_tile) {
  const int lane = threadIdx.x & 31;
  int reach = 0, tiles = 0;                    // carried from one chunk of 32 groups to the next
  for (int g0 = 0; g0 < groups; g0 += 32) {
    const int g = g0 + lane;
    int lo, n;
    ragged_chunk(offsets, counts, groups, rows, g, reach, lo, n);
    const int mine = g < groups ? (tile_rows ? (n + tile_rows - 1) / tile_rows : 1) * tiles_per_row_tile : 0;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    if (g < groups) {
      begin[g] = lo;
      count[g] = n;
      first_tile[g] = tiles + upto - mine;
    }
    tiles += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) first_tile[groups] = tiles;
}

// Tile `local` of a group with m_tiles x n_tiles of them: row tiles fastest inside a band of `band` row tiles, so that
// the tiles in flight share few column panels and the band's rows stay in L2 while the panels pass.
__device__ __forceinline__ void ragged_tile(int local, int m_tiles, int n_tiles, int band, int& m, int& n) {
  const int per_band = band * n_tiles;
  const int b = local / per_band;
  const int rem = local - b * per_band;
  const int m0 = b * band;
  const int in_band = min(band, m_tiles - m0);
  n = rem / in_band;
  m = m0 + rem - n * in_band;
}

// Loads and commits of one CTA or of an SM pair; `bar` is an address in the shared::cluster window (a CTA's own
// shared-memory address is one too).
template <bool kPair>
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if constexpr (kPair) tma_load_2d_pair(dst, map, bar, x, y);
  else tma_load_2d(dst, map, bar, x, y);
}
template <bool kPair>
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (kPair) tma_load_3d_pair(dst, map, bar, x, y, z);
  else tma_load_3d(dst, map, bar, x, y, z);
}
template <bool kPair>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (kPair) umma_commit_both(bar);
  else umma_commit(bar);
}

// One warp's tile of 32 rows x 64 bytes: lane l has written row l as four 16-byte pieces at `store_piece` places.
__device__ __forceinline__ uint32_t store_piece(int row, int piece) {
  return row * kStoreRowBytes + ((piece ^ ((row >> 1) & 3)) << 4);
}

// The sums of a 128 x 128 tile whose contraction the `split` CTAs of a cluster have shared.  A warp of each CTA's eight holds
// rows quarter * 32 + lane and 16 quadruples of columns, quad(j) = columns half * 64 + 4 j .. + 3.  Every CTA lays its sums
// out as [row / 32][column / 4][row % 32][4]; then each of the cluster's warps adds up 64 / split columns of 32 rows, in the
// order of the parts, and hands over eight columns at a time: store(row, column, four, four).  One call per launch: `parts`
// (64 KB) may be what the operands stood in, and `bar` (8 x split arrivals) completes once.
template <typename Quad, typename Store>
__device__ __forceinline__ bool join_parts(uint8_t* parts, uint64_t* bar, int warp, int quarter, int half, int split,
                                           int part, volatile int* abort_ptr, Quad quad, Store store) {
  const int lane = threadIdx.x & 31;
  uint8_t* mine = parts + lane * 16;
#pragma unroll
  for (int j = 0; j < 16; ++j) *reinterpret_cast<float4*>(mine + ((quarter * 32 + half * 16 + j) << 9)) = quad(j);
  __syncwarp();
  if (lane < split) mbar_arrive_cluster(mapa_shared(smem_u32(bar), lane));
  if (!mbar_wait_warp(bar, 0, abort_ptr)) return false;
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
  const int share = warp * 16 + part * 16 / split;         // the first of 16 / split quadruples
  auto finish = [&](auto parts_of) {
    constexpr int kFrom = decltype(parts_of)::value, kQuads = 16 / kFrom;
    float4 v[kFrom][kQuads];
#pragma unroll
    for (int from = 0; from < kFrom; ++from) {
      const uint32_t at = mapa_shared(smem_u32(mine + (share << 9)), from);
#pragma unroll
      for (int j = 0; j < kQuads; ++j) v[from][j] = ld_cluster_f4(at + (j << 9));
    }
#pragma unroll
    for (int from = 1; from < kFrom; ++from)
#pragma unroll
      for (int j = 0; j < kQuads; ++j) {
        v[0][j].x += v[from][j].x; v[0][j].y += v[from][j].y; v[0][j].z += v[from][j].z; v[0][j].w += v[from][j].w;
      }
#pragma unroll
    for (int j = 0; j < kQuads; j += 2) store((share >> 5) * 32 + lane, (share & 31) * 4 + 4 * j, v[0][j], v[0][j + 1]);
  };
  if (split == 8) finish(std::integral_constant<int, 8>{});
  else if (split == 4) finish(std::integral_constant<int, 4>{});
  else finish(std::integral_constant<int, 2>{});
  return true;
}

// Zeros in the rows that belong to no group, dealt to all epilogue warps of the grid.
__device__ __forceinline__ void zero_rows_between(const int* begin, const int* count, int groups, int rows, uint8_t* out,
                                                  long long ld_bytes, int row_bytes, int worker, int workers) {
  const int lane = threadIdx.x & 31;
  int from = 0;
  for (int g = 0; g <= groups; ++g) {
    const int to = g < groups ? begin[g] : rows;
    for (int r = from + worker; r < to; r += workers)
      for (int b = lane * 16; b < row_bytes; b += 512)
        *reinterpret_cast<uint4*>(out + static_cast<long long>(r) * ld_bytes + b) = make_uint4(0, 0, 0, 0);
    if (g < groups) from = begin[g] + count[g];
  }
}

// ------------------------------------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
  static const EncodeTiled fn = []() -> EncodeTiled {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &res) != cudaSuccess ||
        res != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiled>(ptr);
  }();
  return fn;
}

// [groups][rows][cols] with the last dimension contiguous; box of box_rows rows x 128 (swizzle 128) or 64 bytes.  What
// lies past an extent reads as zero and is not written.  groups = 0: a map of two dimensions.
inline int ragged_map(CUtensorMap* map, CUtensorMapDataType type, int elem_bytes, const void* base, int64_t cols,
                      int64_t rows, int64_t groups, int64_t ld, int64_t group_stride, int box_cols, int box_rows) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return COMFY_MOE_EDEVICE;
  if (groups <= 1) group_stride = rows * ld;   // the only one: a stride that is never taken
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(groups)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * elem_bytes, static_cast<cuuint64_t>(group_stride) * elem_bytes};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows), 1u};
  const cuuint32_t one[3] = {1u, 1u, 1u};
  const CUtensorMapSwizzle swizzle = box_cols * elem_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  const CUresult r = encode(map, type, groups ? 3 : 2, const_cast<void*>(base), dims, strides, box, one,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? COMFY_MOE_OK : COMFY_MOE_ECUDA;
}

// Number of SMs of the current device, or a negative value where it is no sm_100.  A thread that has not launched anything
// yet (autograd's, in a backward pass) has no context that the tensor-map encoder could use: cudaSetDevice makes it one.
inline int sm100_count() {
  static thread_local int known = -1, sms = 0;
  int dev = 0, major = 0, count = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -COMFY_MOE_ECUDA;
  if (dev == known) return sms;
  if (cudaSetDevice(dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return -COMFY_MOE_ECUDA;
  known = dev;
  sms = major == 10 ? count : -COMFY_MOE_EDEVICE;
  return sms;
}

// Opts a kernel in to `bytes` of dynamic shared memory, once per thread and device.
template <auto kKernel>
int allow_shared_memory(size_t bytes) {
  static thread_local int done = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return COMFY_MOE_ECUDA;
  if (dev == done) return COMFY_MOE_OK;
  if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != cudaSuccess)
    return COMFY_MOE_ECUDA;
  done = dev;
  return COMFY_MOE_OK;
}

// Sizes whose tiles, row numbers and bytes of a row the kernels count in int32.
inline bool ragged_sizes_fit(int rows, int n, int k) {
  return rows <= COMFY_MOE_RAGGED_MAX_ROWS && n <= COMFY_MOE_RAGGED_MAX_FEATURES && k <= COMFY_MOE_RAGGED_MAX_FEATURES;
}

constexpr size_t ragged_tables(int groups) { return (3 * static_cast<size_t>(groups) + 1) * sizeof(int); }

// Persistent CTAs, one per SM, in clusters of `cluster`; `fixed` bytes of shared memory besides the groups' tables.
template <auto kKernel, typename Params>
int launch_ragged(const Params& p, int threads, size_t fixed, int cluster, int ctas, cudaStream_t stream) {
  const int rc = allow_shared_memory<kKernel>(fixed + ragged_tables(kRaggedMaxGroups) + 1024);
  if (rc != COMFY_MOE_OK) return rc;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = fixed + ragged_tables(p.groups) + 1024;      // (1024: the stages start on a multiple of it)
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kKernel, p) == cudaSuccess ? check_launch() : COMFY_MOE_ECUDA;
}

// Clusters of `size` CTAs of a kernel that the current device holds at once.
template <auto kKernel>
int resident_clusters(int size, int threads, size_t fixed) {
  static thread_local int known = -1, held[9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev != known) {
    const size_t bytes = fixed + ragged_tables(kRaggedMaxGroups) + 1024;
    if (allow_shared_memory<kKernel>(bytes) != COMFY_MOE_OK) return 0;
    for (int s = 2; s <= 8; s *= 2) {
      cudaLaunchConfig_t cfg;
      memset(&cfg, 0, sizeof(cfg));
      cfg.gridDim = dim3(s);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = bytes;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = s;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&held[s], kKernel, &cfg) != cudaSuccess) { cudaGetLastError(); held[s] = 0; }
    }
    known = dev;
  }
  return held[size];
}

// How many CTAs of a cluster share the contraction of each of (at most) `tiles` 128 x 128 tiles; 1: none.  The exchange takes
// 3 us, so a contraction of fewer than `worth` steps is not shared, and no CTA takes fewer than 4.  All clusters have to be
// on the device at once (of 8 CTAs it holds 15): a second wave takes as long as the first.
template <auto kKernel>
int pick_split(int64_t tiles, int64_t steps, int64_t worth, int threads, size_t fixed) {
  if (steps >= worth)
    for (int s = 8; s > 1; s /= 2)
      if (steps >= 4 * s && tiles <= resident_clusters<kKernel>(s, threads, fixed)) return s;
  return 1;
}

inline int64_t up_to(int64_t n, int64_t step) { return (n + step - 1) / step; }

// Rounds of tiles of `tile` rows that the SMs go through, `ctas` of them to a tile, by how many row tiles are to be expected:
// a group's last one is half full, more or less, and no more groups than rows have any.
inline int64_t tile_rounds(int64_t rows, int64_t groups, int64_t tile, int64_t col_tiles, int ctas, int sms) {
  const int64_t busy = groups < rows ? groups : rows, some = rows / tile + busy / 2;
  const int64_t row_tiles = groups == 1 ? up_to(rows, tile) : (some > busy ? some : busy);
  return up_to(row_tiles * col_tiles * ctas, sms);
}

// No more row tiles than these, however the rows are dealt to the groups.
inline int64_t most_row_tiles(int64_t rows, int64_t groups, int64_t tile) {
  return rows / tile + (groups < rows ? groups : rows);
}

}  // namespace comfy_b200
