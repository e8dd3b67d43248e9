// e4m3 matrix products with a scale for each block of 128 along the contraction, dense or grouped by expert, on tcgen05:
//   out[r, n] = sum over blocks b of  xs[r, b] ws[g][n / 128, b]  (sum over k in b of xq[r, k] wq[g][n, k])   (+ bias[n])
// and the same with the weight transposed (the gradient of x: the contraction runs over n, and the 128 x 128 blocks
// transpose with the weight).  A stage of shared memory is one block of the contraction: 128 bytes per row.  The scales
// change with every block, so a block's products cannot stay in one accumulator: the MMAs of a block write a TMEM buffer
// of 128 x 128 per CTA, one of four, and the epilogue warps fold it into sums in registers, one FMA per element and block
// with the product of the two scales.  Every rounding is fp32 until the last one.
// What bounds it is the hand-over between the MMA warp and the epilogue: a wait costs either side 150 cycles even on a
// complete barrier, a block's MMAs take 256, and a way from one CTA of a pair to the other some hundred.  So two blocks
// share a stage, a wait, a commit and a hand-over: 8192 rows, 2560 -> 6912 took 194 us with one block at a time and takes
// 156 (without the quantiser; 1860 TFLOP/s).  Arrivals at the leader with release semantics, which such a barrier does not
// need (what it hands back is tensor memory whose reads are complete), cost a thousand cycles each: 300 us.
// Group rows, tile order and stores as in grouped_matmul_sm100.cu.
#include "few_rows.cuh"
#include "ragged.cuh"

namespace comfy_b200 {

constexpr int kBlk = COMFY_MOE_SCALE_BLOCK;      // elements per scale = bytes per row of a stage
constexpr int kFpTile = 128;                     // rows and columns of a CTA's accumulator, and columns of a tile
constexpr int kFpOperand = kFpTile * kBlk;       // 16 KB
constexpr int kFpUnit = 2;                       // blocks of the contraction per stage, and accumulators per hand-over
constexpr int kFpAcc = 2;                        // pairs of accumulators
constexpr int kFpTmemCols = kFpAcc * kFpUnit * kFpTile;
constexpr int kScaleSteps = 8, kScaleSlots = 2;  // blocks per slot of the ring of scales, slots
constexpr int kScaleWarps = 2;
constexpr int kFpFirst = 2 + kScaleWarps;        // the first epilogue warp
constexpr int kFpThreads = (kFpFirst + kRaggedEpilogueWarps) * 32;
// Registers: the epilogue's two warpgroups hold 64 sums and two steps' 128 products per thread; the first warpgroup
// (producer, MMA issuer, scales) hands over what it does not use.
constexpr int kFpFewRegs = 56, kFpManyRegs = 224, kFpLaunchRegs = 168;
static_assert(kFpThreads == 384 && 128 * kFpFewRegs + 256 * kFpManyRegs <= kFpThreads * kFpLaunchRegs,
              "the warpgroups share what the block is launched with");
static_assert(kBlk == 128, "a stage row is one scale block and one swizzled line");

// kCtas = 1: 128 x 128 tiles.  kCtas = 2: SM pairs, 256 x 128 tiles; each CTA loads its 128 rows and 64 of the columns.
template <int kCtas> struct FpShape {
  static constexpr int kTileRows = kFpTile * kCtas;
  static constexpr int kCols = kFpTile / kCtas;  // columns that a CTA loads
  static constexpr int kBBytes = kCols * kBlk;   // of one block
  static constexpr int kStageBytes = kFpUnit * (kFpOperand + kBBytes);
  static constexpr int kStages = 3;
  static constexpr int kStoreTiles = kCtas;      // of an epilogue warp: pairs have room to store both halves without a wait between
  static constexpr int kStoreBytes = kStoreTiles * kStoreTileBytes;
  static constexpr int kScales = kStages * kStageBytes + kRaggedEpilogueWarps * kStoreBytes;
  static constexpr int kTables = kScales + kScaleSlots * kScaleSteps * kFpTile * 4;
  static_assert(kStages > kFpAcc, "a stage's barriers are never a whole turn ahead of an epilogue warp");
};

__device__ __forceinline__ void unpack_8(const uint4& raw, bool fp16, float (&f)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 v = fp16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[j]))
                          : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
    f[2 * j] = v.x;
    f[2 * j + 1] = v.y;
  }
}

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
  int split;                                     // CTAs that share a tile's contraction (kSplit)
  uint32_t idesc;
};

template <bool kTransposed, int kCtas, bool kSplit>
__global__ void __launch_bounds__(kFpThreads, 1) block_matmul_kernel(const __grid_constant__ BlockParams p) {
  using Shape = FpShape<kCtas>;
  constexpr bool kPair = kCtas == 2;
  static_assert(!kPair || !kSplit, "a contraction is split among single CTAs");
  constexpr int kStages = Shape::kStages, kStageBytes = Shape::kStageBytes, kTileRows = Shape::kTileRows;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages];
  __shared__ __align__(8) uint64_t scale_full_bar[kScaleSlots], scale_empty_bar[kScaleSlots], drain_bar, parts_bar;
  __shared__ int4 tile_ring[kScaleSlots];          // of the slot's tile: first row and column, rows and first row of its group
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? static_cast<int>(cluster_ctarank()) : 0;      // 0 = leader of the pair
  const int split = kSplit ? p.split : 1, part = kSplit ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / (kCtas * split), units = gridDim.x / (kCtas * split);
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* s_begin = reinterpret_cast<int*>(smem + Shape::kTables);
  int* s_count = s_begin + p.groups;
  int* s_first = s_count + p.groups;
  const int n_tiles = (p.n_total + kFpTile - 1) / kFpTile;
  const int blocks = (p.k_total + kBlk - 1) / kBlk, turns = (blocks + kFpUnit - 1) / kFpUnit;
  const int first = kSplit ? turns * part / split * kFpUnit : 0;      // blocks first .. steps - 1 are this CTA's
  const int steps = kSplit ? min(turns * (part + 1) / split * kFpUnit, blocks) : blocks;
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kStages; ++s) { mbar_init(&full_bar[s], 1 + kRaggedEpilogueWarps * kCtas); mbar_init(&empty_bar[s], 1); }
      for (int s = 0; s < kScaleSlots; ++s) { mbar_init(&scale_full_bar[s], kScaleWarps); mbar_init(&scale_empty_bar[s], kRaggedEpilogueWarps); }
      mbar_init(&drain_bar, 1);
      mbar_init(&parts_bar, kRaggedEpilogueWarps * split);
      fence_mbar_init();
      abort_flag = 0;
    }
    __syncwarp();
    ragged_ranges(p.offsets, p.counts, p.groups, p.rows, kTileRows, n_tiles, s_begin, s_count, s_first);
  } else if (warp == 1) {
    if constexpr (kPair) { tmem_alloc_pair(&tmem_slot, kFpTmemCols); tmem_relinquish_pair(); }
    else { tmem_alloc(&tmem_slot, kFpTmemCols); tmem_relinquish(); }
  }
  __syncwarp();
  tc_fence_before_sync();
  if constexpr (kPair || kSplit) cluster_sync_all();     // the peers' barriers must exist before anything signals them
  else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  volatile int* abort_ptr = &abort_flag;
  const int total = kSplit ? min(s_first[p.groups], unit + 1) : s_first[p.groups];      // (clusters: one tile each)
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
    ragged_tile(t - s_first[g], (c.count + kTileRows - 1) / kTileRows, n_tiles, p.band, m, n);
    c.m0 = m * kTileRows;
    c.n0 = n * kFpTile;
    return c;
  };

  float* scale_ring = reinterpret_cast<float*>(smem + Shape::kScales);      // [slot][step][row]
  // Barriers: full[s] is complete when the stage's operands have landed AND every epilogue warp of the tile has read the
  // accumulators that its MMAs will overwrite (they arrive kFpAcc stages ahead), and empty[s], which the MMAs complete, tells
  // the producer that the stage is free and the epilogue that its accumulators are full.
  if (warp < kFpFirst) {
    regs_down<kFpFewRegs>();
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      int s = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int t = unit, g = 0; t < total && ok; t += units) {
        const Tile c = tile_at(t, g);
        for (int kb = first; kb < steps; kb += kFpUnit) {
          ok = mbar_wait_warp(&empty_bar[s], phase, abort_ptr);
          if (!ok) { give_up(kStatusRaggedProducer); break; }
          uint8_t* a = smem + s * kStageBytes;
          uint8_t* b = a + kFpUnit * kFpOperand;
          if (elect_one()) {
            if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], kCtas * kStageBytes);
            const uint32_t bar = kPair ? mapa_shared(smem_u32(&full_bar[s]), 0) : smem_u32(&full_bar[s]);
            const int n0 = c.n0 + rank * Shape::kCols;
#pragma unroll
            for (int u = 0; u < kFpUnit; ++u) {          // (a block behind the last one reads as zeros)
              const int k0 = (kb + u) * kBlk;
              load_2d<kPair>(a + u * kFpOperand, &p.map_a, bar, k0, c.begin + c.m0 + rank * kFpTile);
              load_3d<kPair>(b + u * Shape::kBBytes, &p.map_b, bar, kTransposed ? n0 : k0, kTransposed ? k0 : n0, g);
            }
          }
          __syncwarp();
          s = s + 1 == kStages ? 0 : s + 1;
          phase ^= s == 0;
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer (of the leader)
      int s = 0, acc = 0;
      uint32_t phase = 0;
      const uint32_t a_addr = smem_u32(smem), b_addr = a_addr + kFpUnit * kFpOperand;
      const uint64_t a_first = umma_desc_k_sw128(a_addr);
      const uint64_t b_first = kTransposed ? (kPair ? umma_desc_mn_sw64(b_addr) : umma_desc_mn_sw128(b_addr, kFpOperand))
                                           : umma_desc_k_sw128(b_addr);
      bool ok = true;
      for (int t = unit; t < total && ok && rank == 0; t += units) {
        for (int kb = first; kb < steps; kb += kFpUnit) {
          ok = mbar_wait_warp(&full_bar[s], phase, abort_ptr);
          if (!ok) { give_up(kStatusRaggedMma); break; }
          tc_fence_after_sync();
          if (elect_one()) {
            // 32 steps of the contraction per MMA: 32 bytes along a K-major row, 32 rows of an MN-major box
            constexpr uint32_t kAdvB = kTransposed ? (32 * Shape::kCols) >> 4 : 2;
            const uint64_t a_desc = a_first + s * (kStageBytes >> 4), b_desc = b_first + s * (kStageBytes >> 4);
#pragma unroll
            for (int u = 0; u < kFpUnit; ++u) {
              const uint32_t d_tmem = tmem_base + (acc * kFpUnit + u) * kFpTile;
#pragma unroll
              for (int k = 0; k < kBlk / 32; ++k) {
                const uint64_t ad = a_desc + u * (kFpOperand >> 4) + 2 * k, bd = b_desc + u * (Shape::kBBytes >> 4) + k * kAdvB;
                if constexpr (kPair) umma_ss_pair<true>(d_tmem, ad, bd, p.idesc, k != 0 ? 1u : 0u);
                else umma_ss<true>(d_tmem, ad, bd, p.idesc, k != 0 ? 1u : 0u);
              }
            }
            commit<kPair>(&empty_bar[s]);
          }
          __syncwarp();
          acc = (acc + 1) % kFpAcc;
          s = s + 1 == kStages ? 0 : s + 1;
          phase ^= s == 0;
        }
      }
      if (rank == 0) {                                // nothing of this warp is still running when TMEM is released
        if (elect_one()) {
          if constexpr (kPair) umma_commit_pair(mapa_shared(smem_u32(&drain_bar), 0));
          else umma_commit(&drain_bar);
        }
        __syncwarp();
        mbar_wait(&drain_bar, 0, abort_ptr);
      }
    } else {
      // ------------------------------------------------------------------ scales: xs[row, block] ws[column block, block]
      // One slot holds eight steps of a tile's 128 rows of this CTA.  These warps run ahead of the epilogue, across tiles, so
      // that nobody waits for a load from global memory, which takes longer than a step.
      uint32_t slot = 0;
      bool ok = true;
      for (int t = unit, g = 0; t < total && ok; t += units) {
        const Tile c = tile_at(t, g);
        const float* ws = p.ws + g * p.ws_group + static_cast<long long>(c.n0 / kBlk) * p.ws_n;
        for (int kb = first; kb < steps; kb += kScaleSteps, ++slot) {
          const int q = slot % kScaleSlots;
          ok = mbar_wait_warp(&scale_empty_bar[q], ((slot / kScaleSlots) & 1u) ^ 1u, abort_ptr);
          if (!ok) { give_up(kStatusRaggedEpilogue); break; }
          float w[kScaleSteps];
#pragma unroll
          for (int i = 0; i < kScaleSteps; ++i) w[i] = kb + i < steps ? __ldg(ws + static_cast<long long>(kb + i) * p.ws_k) : 0.f;
#pragma unroll
          for (int v = 0; v < kFpTile / (32 * kScaleWarps); ++v) {
            const int row = ((warp - 2) + v * kScaleWarps) * 32 + lane;
            const int in_group = c.m0 + rank * kFpTile + row;
            const float* xs = p.xs + c.begin + in_group;
            float x[kScaleSteps];
#pragma unroll
            for (int i = 0; i < kScaleSteps; ++i)
              x[i] = kb + i < steps && in_group < c.count ? __ldg(xs + (kb + i) * p.ld_xs) : 0.f;
#pragma unroll
            for (int i = 0; i < kScaleSteps; ++i) scale_ring[(q * kScaleSteps + i) * kFpTile + row] = x[i] * w[i];
          }
          if (warp == 2 && lane == 0) tile_ring[q] = make_int4(c.m0, c.n0, c.count, c.begin);
          __syncwarp();
          if (lane == 0) mbar_arrive(&scale_full_bar[q]);
        }
      }
    }
  } else {
    regs_up<kFpManyRegs>();
    // ------------------------------------------------------------------ epilogue: one row and half of the columns per thread
    const int quarter = warp & 3, half = (warp - kFpFirst) >> 2;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * 64;
    uint8_t* store = smem + kStages * kStageBytes + (warp - kFpFirst) * Shape::kStoreBytes;
    const uint32_t full_addr = kPair ? mapa_shared(smem_u32(full_bar), 0) : smem_u32(full_bar);
    int back = 0;                                // stage of the step whose accumulator is handed back next
    auto hand_back = [&]() {
      if (lane == 0) {
        if constexpr (kPair) mbar_arrive_cluster_relaxed(full_addr + 8 * back);
        else mbar_arrive(&full_bar[back]);
      }
      back = back + 1 == kStages ? 0 : back + 1;
    };
#pragma unroll
    for (int i = 0; i < kFpAcc; ++i) hand_back();     // the first steps find their accumulators free
    int stage = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0, acc_addr = lane_base;      // (accumulators alternate: TMEM's columns begin at 0)
    bool ok = true;
    for (int t = unit; t < total && ok; t += units) {
      float sum[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) sum[i] = 0.f;
      int4 tile = make_int4(0, 0, 0, 0);
      for (int kb = first; kb < steps && ok; kb += kScaleSteps) {
        ok = mbar_wait_warp(&scale_full_bar[slot], slot_phase, abort_ptr);
        if (!ok) { give_up(kStatusRaggedEpilogue); break; }
        const float* scales = scale_ring + slot * kScaleSteps * kFpTile + quarter * 32 + lane;
        tile = tile_ring[slot];
#pragma unroll
        for (int v = 0; v < kScaleSteps; v += kFpUnit) {
          if (kb + v >= steps) break;
          ok = mbar_wait_warp(&empty_bar[stage], phase, abort_ptr);
          if (!ok) { give_up(kStatusRaggedEpilogue); break; }
          stage = stage + 1 == kStages ? 0 : stage + 1;
          phase ^= stage == 0;
          tc_fence_after_sync();
          uint32_t r[kFpUnit][2][32];
          float scale[kFpUnit];
#pragma unroll
          for (int u = 0; u < kFpUnit; ++u) {
            tmem_ld_32x32b_x32(acc_addr + u * kFpTile, r[u][0]);
            tmem_ld_32x32b_x32(acc_addr + u * kFpTile + 32, r[u][1]);
            scale[u] = scales[(v + u) * kFpTile];
          }
          acc_addr ^= kFpUnit * kFpTile;
          tmem_ld_wait();
          tc_fence_before_sync();
          __syncwarp();
          hand_back();
#pragma unroll
          for (int u = 0; u < kFpUnit; ++u)
#pragma unroll
            for (int j = 0; j < 64; ++j) sum[j] = fmaf(__uint_as_float(r[u][j >> 5][j & 31]), scale[u], sum[j]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&scale_empty_bar[slot]);
        slot = slot + 1 == kScaleSlots ? 0 : slot + 1;
        slot_phase ^= slot == 0;
      }
      if (!ok) break;
      if constexpr (kSplit) {
        ok = join_parts(
            smem, &parts_bar, warp - kFpFirst, quarter, half, split, part, abort_ptr,
            [&](int j) { return make_float4(sum[4 * j], sum[4 * j + 1], sum[4 * j + 2], sum[4 * j + 3]); },
            [&](int row, int col, float4 a, float4 b) {
              row += tile.x;
              col += tile.y;
              if (row >= tile.z || col >= p.n_total) return;
              if (p.bias != nullptr) {
                float f[8];
                unpack_8(__ldg(reinterpret_cast<const uint4*>(p.bias) + col / 8), p.fp16, f);
                a.x += f[0]; a.y += f[1]; a.z += f[2]; a.w += f[3];
                b.x += f[4]; b.y += f[5]; b.z += f[6]; b.w += f[7];
              }
              *reinterpret_cast<uint4*>(p.out + (tile.w + row) * p.ld_out + 2 * col) = pack_8(a, b, p.fp16);
            });
        if (!ok) { give_up(kStatusRaggedEpilogue); break; }
        continue;
      }
      const int row0 = tile.x + rank * kFpTile + quarter * 32, rows_here = tile.z - row0;
      if (rows_here <= 0) continue;
      const int col0 = tile.y + half * 64;
      if (p.bias != nullptr) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (col0 + q * 8 >= p.n_total) break;
          float f[8];
          unpack_8(__ldg(reinterpret_cast<const uint4*>(p.bias) + col0 / 8 + q), p.fp16, f);
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[q * 8 + j] += f[j];
        }
      }
      uint32_t packed[32];
      if (p.fp16) {
#pragma unroll
        for (int j = 0; j < 32; ++j) packed[j] = pack_f16x2(sum[2 * j], sum[2 * j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) packed[j] = pack_bf16x2(sum[2 * j], sum[2 * j + 1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = col0 + i * 32;
        if (col >= p.n_total) break;
        uint8_t* store_i = store + i % Shape::kStoreTiles * kStoreTileBytes;
        if (i % Shape::kStoreTiles == 0) {
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(store_i + store_piece(lane, q)) =
              make_uint4(packed[i * 16 + q * 4], packed[i * 16 + q * 4 + 1], packed[i * 16 + q * 4 + 2], packed[i * 16 + q * 4 + 3]);
        if (rows_here >= 32) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.map_out, store_i, col, tile.w + row0);
            bulk_commit_group();
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = k * 8 + (lane >> 2), piece = lane & 3;
            if (row < rows_here && col + piece * 8 < p.n_total)
              *reinterpret_cast<uint4*>(p.out + static_cast<long long>(tile.w + row0 + row) * p.ld_out + 2 * (col + piece * 8)) =
                  *reinterpret_cast<const uint4*>(store_i + store_piece(row, piece));
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    if (p.zero_unused)
      zero_rows_between(s_begin, s_count, p.groups, p.rows, p.out, p.ld_out, 2 * p.n_total,
                        blockIdx.x * kRaggedEpilogueWarps + warp - kFpFirst, gridDim.x * kRaggedEpilogueWarps);
  }

  // ------------------------------------------------------------------ teardown
  __syncwarp();
  if (*abort_ptr) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) __nanosleep(1000);     // copies in flight may still land in shared memory
  }
  tc_fence_before_sync();
  if constexpr (kPair || kSplit) cluster_sync_all();      // no CTA leaves while another may still signal it or read from it
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (kPair) tmem_dealloc_pair(tmem_base, kFpTmemCols);
    else tmem_dealloc(tmem_base, kFpTmemCols);
  }
}

template <bool kTransposed, int kCtas, bool kSplit>
static int launch_block(const BlockParams& p, int cluster, int ctas, cudaStream_t stream) {
  // the warpgroups' register shares have to be there at launch, or the larger ones would wait for good
  static const int regs = [] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, block_matmul_kernel<kTransposed, kCtas, kSplit>) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs < kFpLaunchRegs) return COMFY_MOE_EUNSUPPORTED;
  return launch_ragged<block_matmul_kernel<kTransposed, kCtas, kSplit>>(p, kFpThreads, FpShape<kCtas>::kTables, cluster, ctas,
                                                                        stream);
}

template <bool kTransposed>
static int launch_block_plan(const BlockParams& p, int ctas, int tiles, int sms, cudaStream_t stream) {
  if (p.split > 1) return launch_block<kTransposed, 1, true>(p, p.split, tiles * p.split, stream);
  return ctas == 2 ? launch_block<kTransposed, 2, false>(p, 2, sms / 2 * 2, stream)
                   : launch_block<kTransposed, 1, false>(p, 1, sms, stream);
}

// Blocks from which on the contraction of few tiles is shared by clusters (pick_split).  Measured (us, whole / shared): 100
// rows, 8192 -> 256: 22.8 / 12.9; 64 rows, 6912 -> 2560: 20.6 / 14.2; with 20 blocks, 2560 -> 2560: 12.7 / 12.0.
constexpr int kSplitBlocks = 20;

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
  if (n_groups > kRaggedMaxGroups || k % 16 || in % 16 || cols % 8 || !ragged_sizes_fit(rows, n, k)) return COMFY_MOE_EUNSUPPORTED;
  if (n_groups != 1 && !offsets) return COMFY_MOE_EINVAL;
  if (rows == 0) return COMFY_MOE_OK;
  const bool quantise_inside = !transpose_w && rows <= kFewRowsQuantise && k <= kFewQuantiseMaxK;
  if (!x || (!workspace && !quantise_inside) || !out || !aligned16(x) || !aligned16(workspace) || !aligned16(out) || ld_x < in || ld_x % 8 ||
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
  const int nb = (n + kBlk - 1) / kBlk, kb = (k + kBlk - 1) / kBlk;
  uint8_t* q = static_cast<uint8_t*>(workspace);
  float* xs = quantise_inside ? nullptr : reinterpret_cast<float*>(q + scale_offset(rows, in));
  int rc = quantise_inside ? COMFY_MOE_OK : comfy_moe_block_quantize(x, ld_x, dtype, rows, in, q, in, xs, rows, stream);
  if (rc != COMFY_MOE_OK) return rc;
  if (!transpose_w && rows <= kFewRowsBlock) {
    FewParams f;
    memset(&f, 0, sizeof(f));
    f.x = quantise_inside ? static_cast<const uint8_t*>(x) : q;
    f.ld_x = quantise_inside ? ld_x * 2 : in;
    f.xs = xs; f.ld_xs = rows;
    f.w = static_cast<const uint8_t*>(w); f.out = static_cast<uint8_t*>(out);
    f.offsets = offsets; f.counts = counts;
    f.ws = w_scale; f.ws_group = static_cast<long long>(nb) * kb;
    f.bias = bias;
    f.ld_w = ld_w; f.w_group = w_group_stride; f.ld_out = ld_out * 2;
    f.groups = n_groups; f.rows = rows; f.n = n; f.k = k; f.zero_unused = zero_unused;
    return launch_few_rows_block(f, dtype == COMFY_MOE_FP16, s);
  }
  const int64_t col_tiles = up_to(cols, kFpTile), tiles = most_row_tiles(rows, n_groups, kFpTile) * col_tiles;
  const int split = pick_split<block_matmul_kernel<false, 1, true>>(tiles, (in + kBlk - 1) / kBlk, kSplitBlocks, kFpThreads,
                                                                    FpShape<1>::kTables);
  // A step of a pair's 256 x 128 tile takes 6 % less than one of a single CTA's 128 x 128, but half-empty row tiles may add
  // rounds (us, pair / single): one group, 2560 -> 6912: 1999 rows 47.8 / 50.6; 4 groups: 500 rows each, 8 and 7 rounds,
  // 61.9 / 58.2; 1400, 18 and 17, 123.7 / 131.8; 8 groups, 1008 -> 2064, the gradient at 200 rows, 2 and 1: 25.0 / 18.5.
  const bool pairs = 16 * tile_rounds(rows, n_groups, 2 * kFpTile, col_tiles, 2, sms) <=
                     17 * tile_rounds(rows, n_groups, kFpTile, col_tiles, 1, sms);
  const int ctas = split == 1 && pairs ? 2 : 1;
  BlockParams p;
  memset(&p, 0, sizeof(p));
  const CUtensorMapDataType t = dtype == COMFY_MOE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if ((rc = ragged_map(&p.map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q, in, rows, 0, in, 0, kBlk, kFpTile)) != COMFY_MOE_OK ||
      (rc = ragged_map(&p.map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, k, n, n_groups, ld_w, w_group_stride,
                       transpose_w ? kFpTile / ctas : kBlk, transpose_w ? kBlk : kFpTile / ctas)) != COMFY_MOE_OK ||
      (rc = ragged_map(&p.map_out, t, 2, out, cols, rows, 0, ld_out, 0, 32, 32)) != COMFY_MOE_OK)
    return rc;
  p.offsets = offsets; p.counts = counts;
  p.xs = xs; p.ld_xs = rows;
  p.ws = w_scale; p.ws_group = static_cast<long long>(nb) * kb;
  p.ws_n = transpose_w ? 1 : kb;
  p.ws_k = transpose_w ? kb : 1;
  p.bias = bias;
  p.out = static_cast<uint8_t*>(out); p.ld_out = ld_out * 2;
  p.status = status;
  p.groups = n_groups; p.rows = rows; p.n_total = cols; p.k_total = in;
  p.zero_unused = zero_unused;
  p.fp16 = dtype == COMFY_MOE_FP16;
  const int64_t band = (32ll << 20) / (static_cast<int64_t>(kFpTile * ctas) * in);   // 32 MB of rows stay in L2
  p.band = static_cast<int>(band < 8 ? 8 : (band > 64 ? 64 : band));
  p.idesc = umma_idesc<true>(kFpTile * ctas, kFpTile) | (transpose_w ? 1u << 16 : 0u);
  p.split = split;
  return transpose_w ? launch_block_plan<true>(p, ctas, static_cast<int>(tiles), sms, s)
                     : launch_block_plan<false>(p, ctas, static_cast<int>(tiles), sms, s);
}
