// e4m3 matrix products with a scale for each block of 128 along the contraction, dense or grouped by expert, on tcgen05:
//   out[r, n] = sum over blocks b of  xs[r, b] ws[g][n / 128, b]  (sum over k in b of xq[r, k] wq[g][n, k])   (+ bias[n])
// and the same with the weight transposed (the gradient of x: the contraction runs over n, and the 128 x 128 blocks
// transpose with the weight).  A stage of shared memory is one block of the contraction: 128 bytes per row.  The scales
// change with every block, so a block's 128 x 128 products cannot stay in one accumulator: the MMAs of a block write a
// TMEM buffer of their own (four of them in flight), and the epilogue warps fold it into sums in registers, one FMA per
// element and block with the product of the two scales.  Every rounding is fp32 until the last one.
// Group rows, tile order and stores as in grouped_matmul_sm100.cu.
#include "ragged.cuh"

namespace comfy_b200 {

constexpr int kBlk = COMFY_MOE_SCALE_BLOCK;      // elements per scale = bytes per row of a stage
constexpr int kFpTile = 128;                     // rows and columns of a tile
constexpr int kFpOperand = kFpTile * kBlk;       // 16 KB
constexpr int kFpStageBytes = 2 * kFpOperand;
constexpr int kFpStages = 6;
constexpr int kFpAcc = 4;                        // TMEM buffers of 128 columns
constexpr int kFpTables = kFpStages * kFpStageBytes + kRaggedEpilogueWarps * kStoreTileBytes;
static_assert(kBlk == 128, "a stage row is one scale block and one swizzled line");

struct alignas(64) BlockParams {
  CUtensorMap map_a, map_b, map_out;
  const int32_t* offsets;
  const int32_t* counts;
  const float* xs;                               // [blocks][ld_xs]
  const float* ws;
  const void* bias;
  uint8_t* out;
  int32_t* status;
  long long ld_out;                              // bytes
  long long ld_xs;
  long long ws_group;                            // scales per group
  int ws_n, ws_k;                                // strides over column blocks and contraction blocks
  int groups, rows, n_total, k_total, band, zero_unused, fp16;
  uint32_t idesc;
};

template <bool kTransposed>
__global__ void __launch_bounds__(kRaggedThreads, 1) block_matmul_kernel(const __grid_constant__ BlockParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kFpStages], empty_bar[kFpStages];
  __shared__ __align__(8) uint64_t tmem_full_bar[kFpAcc], tmem_empty_bar[kFpAcc], drain_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* s_begin = reinterpret_cast<int*>(smem + kFpTables);
  int* s_count = s_begin + p.groups;
  int* s_first = s_count + p.groups;
  const int n_tiles = (p.n_total + kFpTile - 1) / kFpTile;
  const int steps = (p.k_total + kBlk - 1) / kBlk;
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kFpStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
      for (int s = 0; s < kFpAcc; ++s) { mbar_init(&tmem_full_bar[s], 1); mbar_init(&tmem_empty_bar[s], kRaggedEpilogueWarps); }
      mbar_init(&drain_bar, 1);
      fence_mbar_init();
      abort_flag = 0;
    }
    __syncwarp();
    ragged_ranges(p.offsets, p.counts, p.groups, p.rows, kFpTile, n_tiles, s_begin, s_count, s_first);
  } else if (warp == 1) {
    tmem_alloc(&tmem_slot, kFpAcc * kFpTile);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  volatile int* abort_ptr = &abort_flag;
  const int total = s_first[p.groups];
  auto give_up = [&](int code) {
    if (lane == 0) { atomicCAS(p.status, 0, code); abort_flag = 1; }
  };
  struct Tile { int m0, n0, begin, count; };
  auto tile_at = [&](int t, int& g) {
    while (t >= s_first[g + 1]) ++g;
    Tile c;
    c.begin = s_begin[g];
    c.count = s_count[g];
    int m, n;
    ragged_tile(t - s_first[g], (c.count + kFpTile - 1) / kFpTile, n_tiles, p.band, m, n);
    c.m0 = m * kFpTile;
    c.n0 = n * kFpTile;
    return c;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    uint32_t it = 0;
    bool ok = true;
    for (int t = blockIdx.x, g = 0; t < total && ok; t += gridDim.x) {
      const Tile c = tile_at(t, g);
      for (int kb = 0; kb < steps; ++kb, ++it) {
        const int s = it % kFpStages;
        ok = mbar_wait_warp(&empty_bar[s], ((it / kFpStages) & 1u) ^ 1u, abort_ptr);
        if (!ok) { give_up(kStatusRaggedProducer); break; }
        uint8_t* a = smem + s * kFpStageBytes;
        if (elect_one()) {
          mbar_arrive_expect_tx(&full_bar[s], kFpStageBytes);
          tma_load_2d(a, &p.map_a, &full_bar[s], kb * kBlk, c.begin + c.m0);
          if constexpr (kTransposed) tma_load_3d(a + kFpOperand, &p.map_b, &full_bar[s], c.n0, kb * kBlk, g);
          else tma_load_3d(a + kFpOperand, &p.map_b, &full_bar[s], kb * kBlk, c.n0, g);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    uint32_t it = 0;                               // counts stages and, alike, TMEM buffers
    bool ok = true;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      for (int kb = 0; kb < steps; ++kb, ++it) {
        const int s = it % kFpStages, as = it % kFpAcc;
        ok = mbar_wait_warp(&tmem_empty_bar[as], ((it / kFpAcc) & 1u) ^ 1u, abort_ptr) &&
             mbar_wait_warp(&full_bar[s], (it / kFpStages) & 1u, abort_ptr);
        if (!ok) { give_up(kStatusRaggedMma); break; }
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t a_addr = smem_u32(smem + s * kFpStageBytes);
          const uint64_t a_desc = umma_desc_k_sw128(a_addr);
          const uint64_t b_desc = kTransposed ? umma_desc_mn_sw128(a_addr + kFpOperand, kFpOperand)
                                              : umma_desc_k_sw128(a_addr + kFpOperand);
          constexpr uint32_t kAdvB = kTransposed ? (32 * 128) >> 4 : 2;    // 32 steps of the contraction per MMA
#pragma unroll
          for (int k = 0; k < kBlk / 32; ++k)
            umma_ss<true>(tmem_base + as * kFpTile, a_desc + 2 * k, b_desc + k * kAdvB, p.idesc, k != 0 ? 1u : 0u);
          umma_commit(&empty_bar[s]);
          umma_commit(&tmem_full_bar[as]);
        }
        __syncwarp();
      }
    }
    if (elect_one()) umma_commit(&drain_bar);       // nothing of this warp is still running when TMEM is released
    __syncwarp();
    mbar_wait(&drain_bar, 0, abort_ptr);
  } else {
    // ------------------------------------------------------------------ epilogue: one row and 64 columns per thread
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * 64;
    uint8_t* store = smem + kFpStages * kFpStageBytes + (warp - 2) * kStoreTileBytes;
    uint32_t it = 0;
    bool ok = true;
    for (int t = blockIdx.x, g = 0; t < total && ok; t += gridDim.x) {
      const Tile c = tile_at(t, g);
      const int row0 = c.m0 + quarter * 32;
      const int rows_here = c.count - row0;
      const bool live = lane < rows_here;
      const float* xs = p.xs + c.begin + row0 + lane;
      const float* ws = p.ws + g * p.ws_group + static_cast<long long>(c.n0 / kBlk) * p.ws_n;
      float sum[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) sum[i] = 0.f;
      float xs_next = live ? __ldg(xs) : 0.f, ws_next = __ldg(ws);
      for (int kb = 0; kb < steps; ++kb, ++it) {
        const float scale = xs_next * ws_next;
        if (kb + 1 < steps) {
          xs_next = live ? __ldg(xs + (kb + 1) * p.ld_xs) : 0.f;
          ws_next = __ldg(ws + static_cast<long long>(kb + 1) * p.ws_k);
        }
        const uint32_t as = it % kFpAcc;
        ok = mbar_wait_warp(&tmem_full_bar[as], (it / kFpAcc) & 1u, abort_ptr);
        if (!ok) { give_up(kStatusRaggedEpilogue); break; }
        tc_fence_after_sync();
        uint32_t r[2][32];
        tmem_ld_32x32b_x32(lane_base + as * kFpTile, r[0]);
        tmem_ld_32x32b_x32(lane_base + as * kFpTile + 32, r[1]);
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tmem_empty_bar[as]);
#pragma unroll
        for (int i = 0; i < 64; ++i) sum[i] = fmaf(__uint_as_float(r[i >> 5][i & 31]), scale, sum[i]);
      }
      if (!ok || rows_here <= 0) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = c.n0 + half * 64 + i * 32;
        if (col >= p.n_total) continue;
        if (lane == 0) bulk_wait_read_all();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = sum[i * 32 + q * 8 + j];
          if (p.bias != nullptr && col + q * 8 < p.n_total) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p.bias) + (col + q * 8) / 8);
            const uint32_t b[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = p.fp16 ? __half22float2(*reinterpret_cast<const __half2*>(&b[j]))
                                      : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&b[j]));
              v[2 * j] += f.x;
              v[2 * j + 1] += f.y;
            }
          }
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = p.fp16 ? pack_f16x2(v[2 * j], v[2 * j + 1]) : pack_bf16x2(v[2 * j], v[2 * j + 1]);
          *reinterpret_cast<uint4*>(store + store_piece(lane, q)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (rows_here >= 32) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.map_out, store, col, c.begin + row0);
            bulk_commit_group();
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = k * 8 + (lane >> 2), piece = lane & 3;
            if (row < rows_here && col + piece * 8 < p.n_total)
              *reinterpret_cast<uint4*>(p.out + static_cast<long long>(c.begin + row0 + row) * p.ld_out + 2 * (col + piece * 8)) =
                  *reinterpret_cast<const uint4*>(store + store_piece(row, piece));
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    if (p.zero_unused)
      zero_rows_between(s_begin, s_count, p.groups, p.rows, p.out, p.ld_out, 2 * p.n_total,
                        blockIdx.x * kRaggedEpilogueWarps + warp - 2, gridDim.x * kRaggedEpilogueWarps);
  }

  // ------------------------------------------------------------------ teardown
  __syncwarp();
  if (*abort_ptr) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) __nanosleep(1000);     // copies in flight may still land in shared memory
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kFpAcc * kFpTile);
  }
}

template <bool kTransposed>
static int launch_block(const BlockParams& p, int sms, cudaStream_t stream) {
  const size_t smem = kFpTables + (3 * static_cast<size_t>(p.groups) + 1) * sizeof(int) + 1024;
  if (cudaFuncSetAttribute(block_matmul_kernel<kTransposed>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem)) != cudaSuccess)
    return COMFY_MOE_ECUDA;
  block_matmul_kernel<kTransposed><<<sms, kRaggedThreads, smem, stream>>>(p);
  return check_launch();
}

static int64_t scale_offset(int64_t rows, int64_t cols) { return (rows * cols + 255) / 256 * 256; }

}  // namespace comfy_b200

using namespace comfy_b200;

extern "C" int64_t comfy_moe_block_workspace(int rows, int cols) {
  if (rows < 0 || cols < 0) return 0;
  return scale_offset(rows, cols) + static_cast<int64_t>(rows) * ((cols + kBlk - 1) / kBlk) * 4;
}

extern "C" int comfy_moe_block_matmul(const void* x, int64_t ld_x, int dtype, void* workspace, const void* w, int64_t ld_w,
                                      int64_t w_group_stride, const float* w_scale, int transpose_w, int rows, int n_groups,
                                      int out_features, int in_features, const int32_t* offsets, const int32_t* counts,
                                      const void* bias, int zero_unused, void* out, int64_t ld_out, int32_t* status,
                                      void* stream) {
  const int n = out_features, k = in_features;
  if (rows < 0 || n_groups < 0 || n <= 0 || k <= 0 || !status) return COMFY_MOE_EINVAL;
  if (dtype != COMFY_MOE_BF16 && dtype != COMFY_MOE_FP16) return COMFY_MOE_EUNSUPPORTED;
  const int in = transpose_w ? n : k, cols = transpose_w ? k : n;
  if (n_groups > kRaggedMaxGroups || k % 16 || in % 16 || cols % 8) return COMFY_MOE_EUNSUPPORTED;
  if (n_groups != 1 && !offsets) return COMFY_MOE_EINVAL;
  if (rows == 0) return COMFY_MOE_OK;
  if (!x || !workspace || !out || !aligned16(x) || !aligned16(workspace) || !aligned16(out) || ld_x < in || ld_x % 8 ||
      ld_out < cols || ld_out % 8 || (bias && !aligned16(bias)))
    return COMFY_MOE_EINVAL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n_groups == 0) {
    if (zero_unused && cudaMemset2DAsync(out, ld_out * 2, 0, static_cast<size_t>(cols) * 2, rows, s) != cudaSuccess)
      return COMFY_MOE_ECUDA;
    return COMFY_MOE_OK;
  }
  if (!w || !w_scale || !aligned16(w) || ld_w < k || ld_w % 16 || (n_groups > 1 && (w_group_stride <= 0 || w_group_stride % 16)))
    return COMFY_MOE_EINVAL;
  const int sms = sm100_count();
  if (sms < 0) return -sms;
  uint8_t* q = static_cast<uint8_t*>(workspace);
  float* xs = reinterpret_cast<float*>(q + scale_offset(rows, in));
  int rc = comfy_moe_block_quantize(x, ld_x, dtype, rows, in, q, in, xs, rows, stream);
  if (rc != COMFY_MOE_OK) return rc;
  BlockParams p;
  memset(&p, 0, sizeof(p));
  const CUtensorMapDataType t = dtype == COMFY_MOE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if ((rc = ragged_map(&p.map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q, in, rows, 0, in, 0, kBlk, kFpTile)) != COMFY_MOE_OK ||
      (rc = ragged_map(&p.map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, k, n, n_groups, ld_w, w_group_stride, kBlk, kFpTile)) != COMFY_MOE_OK ||
      (rc = ragged_map(&p.map_out, t, 2, out, cols, rows, 0, ld_out, 0, 32, 32)) != COMFY_MOE_OK)
    return rc;
  const int nb = (n + kBlk - 1) / kBlk, kb = (k + kBlk - 1) / kBlk;
  p.offsets = offsets; p.counts = counts;
  p.xs = xs; p.ld_xs = rows;
  p.ws = w_scale; p.ws_group = static_cast<long long>(nb) * kb;
  p.ws_n = transpose_w ? 1 : kb;
  p.ws_k = transpose_w ? kb : 1;
  p.bias = bias;
  p.out = static_cast<uint8_t*>(out); p.ld_out = ld_out * 2;
  p.status = status;
  p.groups = n_groups; p.rows = rows; p.n_total = cols; p.k_total = in;
  const int64_t band = (32ll << 20) / (static_cast<int64_t>(kFpTile) * in);   // 32 MB of rows stay in L2
  p.band = static_cast<int>(band < 8 ? 8 : (band > 64 ? 64 : band));
  p.zero_unused = zero_unused;
  p.fp16 = dtype == COMFY_MOE_FP16;
  p.idesc = umma_idesc<true>(kFpTile, kFpTile) | (transpose_w ? 1u << 16 : 0u);
  return transpose_w ? launch_block<true>(p, sms, s) : launch_block<false>(p, sms, s);
}
