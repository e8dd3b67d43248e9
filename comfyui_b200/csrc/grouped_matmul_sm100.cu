// Matrix products grouped by expert with ragged sizes, and their gradients, on tcgen05 tensor cores:
//   forward   y[r, :]  = x[r, :] W[g]^T                 for the rows r of group g,   x [R, K], W [G, N, K], y [R, N]
//   d x       dx[r, :] = dy[r, :] W[g]
//   d W       dw[g]    = sum over the rows r of g of dy[r, :]^T x[r, :]              (zeros for a group without rows)
// The groups' rows are read from the device (offsets, optional counts), so no call waits for the host.  All three run
// on one kernel; what differs is which dimension of an operand is contiguous in memory.  tcgen05 reads both kinds from
// shared memory (a K-major tile: rows of 64 elements of the contraction; an MN-major tile: 64 output elements per row,
// one row per step of the contraction), so nothing is transposed in memory:
//   forward: A = x (K-major), B = W[g] (K-major);   d x: A = dy (K-major), B = W[g] (MN-major);
//   d W: A = dy, B = x, both MN-major, contraction over the group's rows.
// A row of a tile depends on its own row of A only, so tiles of the first two may hang over the end of their group: the
// loads take what follows, the stores leave it out.  In d W the rows behind the group are part of the sum: a warp of its own
// overwrites them with zeros in shared memory (both operands: what stands there may be NaN) before they are multiplied.
//
// kSplit: a cluster shares each tile's contraction (few tiles, long contraction: plan_gmm).
// kCtas = 2: two CTAs on an SM pair share one tcgen05.mma.cta_group::2 stream.  Their tile is 256 rows x 256 columns; each
// loads its own 128 rows of A and half of B's columns, so an SM reads a third less per product than with 128 x 256 of its
// own, and under the power cap the clock rises by as much.  Barriers as in moe_grouped_gemm_sm100.cu: full and
// tmem_empty live in the leader, both CTAs' loads and epilogue warps signal them; empty and tmem_full exist in both and are
// committed to by the leader's MMA warp.  In d W a group's last, partial step is loaded against a tail barrier of each
// CTA; its tail warp zeroes what lies behind the group and announces the step, in the leader on `full`, in the other CTA on
// the leader's `peer` barrier.  (An arrival of the other CTA at every step, so that one barrier would do, halved the rate:
// 762 us against 412 with single CTAs at 16384 rows, 8 groups, 2048 x 8192.  Zeros by the MMA warp itself held up every
// tile of a short group: 111 us against 108 at 2048 rows.)
#include "few_rows.cuh"
#include "ragged.cuh"

namespace comfy_b200 {

enum RaggedForm { kForward = 0, kGradX = 1, kGradW = 2 };

constexpr int kTileM = 128;
constexpr int kStepK = 64;                     // contraction elements per stage: one 128-byte swizzled row
constexpr int kABytes = kTileM * 128;
constexpr int kMnBoxBytes = kStepK * 128;      // one box of an MN-major operand: 64 steps x 64 elements

constexpr int kStageBytes = 2 * kABytes;        // 128 rows of A, 128 columns of B
constexpr int kStages = 6;
constexpr int kGmmTables = kStages * kStageBytes + kRaggedEpilogueWarps * kStoreTileBytes;

struct alignas(64) GmmParams {
  CUtensorMap map_a, map_b, map_out;
  const int32_t* offsets;
  const int32_t* counts;
  uint8_t* out;
  int32_t* status;
  long long ld_out, out_group;                 // bytes (d W: out_group from one expert to the next)
  int groups, rows;                            // rows of the buffers
  int m_total;                                 // d W: rows of dw[g] (N); otherwise unused
  int n_total;                                 // output columns
  int k_total;                                 // contraction length (d W: the group's rows, unused)
  int band;                                    // row tiles per band of the tile order
  int split;                                   // CTAs that share a tile's contraction (kSplit)
  int zero_unused;
  int fp16, out_fp32;
  uint32_t idesc;
};

template <int kForm, int kCtas, bool kSplit>
__global__ void __launch_bounds__(kForm == kGradW ? kRaggedTailThreads : kRaggedThreads, 1)
grouped_matmul_kernel(const __grid_constant__ GmmParams p) {
  constexpr int kTile = kTileM * kCtas;          // rows and columns
  constexpr int kTmemCols = 2 * kTile;           // two accumulators: the epilogue of one tile overlaps the next one's MMAs
  constexpr bool kPair = kCtas == 2;
  static_assert(!kPair || !kSplit, "a contraction is split among single CTAs");
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages];
  __shared__ __align__(8) uint64_t tmem_full_bar[2], tmem_empty_bar[2], drain_bar;
  __shared__ __align__(8) uint64_t tail_bar[kStages], peer_bar[kStages];
  __shared__ __align__(8) uint64_t parts_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? static_cast<int>(cluster_ctarank()) : 0;      // 0 = leader of the pair
  const int split = kSplit ? p.split : 1, part = kSplit ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / (kCtas * split), units = gridDim.x / (kCtas * split);
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* s_begin = reinterpret_cast<int*>(smem + kGmmTables);
  int* s_count = s_begin + p.groups;
  int* s_first = s_count + p.groups;

  const int n_tiles = (p.n_total + kTile - 1) / kTile;
  const int m_tiles_w = (p.m_total + kTile - 1) / kTile;
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < kStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
      for (int s = 0; s < 2; ++s) { mbar_init(&tmem_full_bar[s], 1); mbar_init(&tmem_empty_bar[s], kRaggedEpilogueWarps * kCtas); }
      mbar_init(&drain_bar, 1);
      for (int s = 0; s < kStages; ++s) { mbar_init(&tail_bar[s], 1); mbar_init(&peer_bar[s], 1); }
      mbar_init(&parts_bar, kRaggedEpilogueWarps * split);
      fence_mbar_init();
      abort_flag = 0;
    }
    __syncwarp();
    ragged_ranges(p.offsets, p.counts, p.groups, p.rows, kForm == kGradW ? 0 : kTile,
                  kForm == kGradW ? m_tiles_w * n_tiles : n_tiles, s_begin, s_count, s_first);
  } else if (warp == 1) {
    if constexpr (kPair) { tmem_alloc_pair(&tmem_slot, kTmemCols); tmem_relinquish_pair(); }
    else { tmem_alloc(&tmem_slot, kTmemCols); tmem_relinquish(); }
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

  // Tiles t = unit, + units, ... in the order of the groups; g only ever moves forward.
  struct Tile { int m0, n0, begin, count, first, steps; };      // steps first .. steps - 1 are this CTA's
  auto tile_at = [&](int t, int& g) {
    while (t >= s_first[g + 1]) ++g;
    Tile c;
    c.begin = s_begin[g];
    c.count = s_count[g];
    int m, n;
    ragged_tile(t - s_first[g], kForm == kGradW ? m_tiles_w : (c.count + kTile - 1) / kTile, n_tiles, p.band, m, n);
    c.m0 = m * kTile;
    c.n0 = n * kTile;
    c.first = 0;
    c.steps = ((kForm == kGradW ? c.count : p.k_total) + kStepK - 1) / kStepK;
    if constexpr (kSplit) {
      c.first = c.steps * part / split;
      c.steps = c.steps * (part + 1) / split;
    }
    return c;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    uint32_t it = 0;
    bool ok = true;
    for (int t = unit, g = 0; t < total && ok; t += units) {
      const Tile c = tile_at(t, g);
      for (int kb = c.first; kb < c.steps; ++kb, ++it) {
        const int s = it % kStages;
        ok = mbar_wait_warp(&empty_bar[s], ((it / kStages) & 1u) ^ 1u, abort_ptr);
        if (!ok) { give_up(kStatusRaggedProducer); break; }
        uint8_t* a = smem + s * kStageBytes;
        uint8_t* b = a + kABytes;
        if (elect_one()) {
          // a step is full in the leader, with both CTAs' bytes; a partial step of d W in each CTA by itself
          const bool tail = kForm == kGradW && c.count - kb * kStepK < kStepK;
          uint64_t* own = tail ? &tail_bar[s] : &full_bar[s];
          if (tail || rank == 0) mbar_arrive_expect_tx(own, tail ? kStageBytes : kCtas * kStageBytes);
          const uint32_t bar = kPair ? mapa_shared(smem_u32(own), tail ? rank : 0) : smem_u32(own);
          const int m0 = c.m0 + rank * kTileM, n0 = c.n0 + rank * kTileM;
          if constexpr (kForm == kGradW) {
#pragma unroll
            for (int i = 0; i < kTileM / 64; ++i)
              load_2d<kPair>(a + i * kMnBoxBytes, &p.map_a, bar, m0 + i * 64, c.begin + kb * kStepK);
#pragma unroll
            for (int i = 0; i < kTileM / 64; ++i)
              load_2d<kPair>(b + i * kMnBoxBytes, &p.map_b, bar, n0 + i * 64, c.begin + kb * kStepK);
          } else {
            load_2d<kPair>(a, &p.map_a, bar, kb * kStepK, c.begin + m0);
            if constexpr (kForm == kForward) {
              load_3d<kPair>(b, &p.map_b, bar, kb * kStepK, n0, g);
            } else {
#pragma unroll
              for (int i = 0; i < kTileM / 64; ++i)
                load_3d<kPair>(b + i * kMnBoxBytes, &p.map_b, bar, n0 + i * 64, kb * kStepK, g);
            }
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (of the leader)
    uint32_t it = 0, acc = 0;
    uint32_t peers = 0;                             // bit s: parity of peer_bar[s]
    bool ok = true;
    for (int t = unit, g = 0; t < total && ok && rank == 0; t += units) {
      const Tile c = tile_at(t, g);
      if (c.steps == c.first) continue;
      const uint32_t as = acc & 1u;
      ok = mbar_wait_warp(&tmem_empty_bar[as], ((acc >> 1) & 1u) ^ 1u, abort_ptr);
      if (!ok) { give_up(kStatusRaggedMma); break; }
      ++acc;
      tc_fence_after_sync();
      const uint32_t d_tmem = tmem_base + as * kTile;
      for (int kb = c.first; kb < c.steps; ++kb, ++it) {
        const int s = it % kStages;
        ok = mbar_wait_warp(&full_bar[s], (it / kStages) & 1u, abort_ptr);
        if (!ok) { give_up(kStatusRaggedMma); break; }
        uint8_t* a = smem + s * kStageBytes;
        if (kForm == kGradW && kPair && c.count - kb * kStepK < kStepK) {
          ok = mbar_wait_warp(&peer_bar[s], (peers >> s) & 1u, abort_ptr);
          if (!ok) { give_up(kStatusRaggedMma); break; }
          peers ^= 1u << s;
          asm volatile("fence.acq_rel.cluster;" ::: "memory");
        }
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t a_addr = smem_u32(a);
          const uint64_t a_desc = kForm == kGradW ? umma_desc_mn_sw128(a_addr, kMnBoxBytes) : umma_desc_k_sw128(a_addr);
          const uint64_t b_desc = kForm == kForward ? umma_desc_k_sw128(a_addr + kABytes)
                                                    : umma_desc_mn_sw128(a_addr + kABytes, kMnBoxBytes);
          // 16 steps of the contraction per MMA: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major box
          constexpr uint32_t kAdvA = kForm == kGradW ? 128 : 2, kAdvB = kForm == kForward ? 2 : 128;
#pragma unroll
          for (int k = 0; k < kStepK / 16; ++k) {
            if constexpr (kPair) umma_ss_pair<false>(d_tmem, a_desc + k * kAdvA, b_desc + k * kAdvB, p.idesc, kb != c.first || k != 0 ? 1u : 0u);
            else umma_ss<false>(d_tmem, a_desc + k * kAdvA, b_desc + k * kAdvB, p.idesc, kb != c.first || k != 0 ? 1u : 0u);
          }
          commit<kPair>(&empty_bar[s]);
        }
        __syncwarp();
      }
      if (ok && elect_one()) commit<kPair>(&tmem_full_bar[as]);
      __syncwarp();
    }
    if (rank == 0) {                                // nothing of this warp is still running when TMEM is released
      if (elect_one()) {
        if constexpr (kPair) umma_commit_pair(mapa_shared(smem_u32(&drain_bar), 0));
        else umma_commit(&drain_bar);
      }
      __syncwarp();
      mbar_wait(&drain_bar, 0, abort_ptr);
    }
  } else if (kForm == kGradW && warp == 2 + kRaggedEpilogueWarps) {
    // ------------------------------------------------------------------ zeros behind a group
    uint32_t it = 0, tails = 0;                     // bit s: parity of tail_bar[s]
    for (int t = unit, g = 0; t < total; t += units) {
      const Tile c = tile_at(t, g);
      it += c.steps - c.first;
      const int valid = c.count - (c.steps - 1) * kStepK;
      if (c.steps == c.first || valid >= kStepK) continue;
      const int s = (it - 1) % kStages;
      if (!mbar_wait_warp(&tail_bar[s], (tails >> s) & 1u, abort_ptr)) { give_up(kStatusRaggedMma); break; }
      tails ^= 1u << s;
      uint8_t* a = smem + s * kStageBytes;
      for (int box = 0; box < 2 * kTileM / 64; ++box)
        for (int o = valid * 128 + lane * 16; o < kMnBoxBytes; o += 512)
          *reinterpret_cast<uint4*>(a + box * kMnBoxBytes + o) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) mbar_arrive(&full_bar[s]);
        else mbar_arrive_cluster(mapa_shared(smem_u32(&peer_bar[s]), 0));
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    uint8_t* store = smem + kStages * kStageBytes + (warp - 2) * kStoreTileBytes;
    // 32 rows from row0 on (inside the group; d W: inside dw[g]) of 32 columns of the output: lane l has row l
    auto emit = [&](const Tile& c, int g, int row0, int col, const uint32_t (&v)[32]) {
      const int rows_here = (kForm == kGradW ? p.m_total : c.count) - row0;
      if (rows_here <= 0 || col >= p.n_total) return;
      const int sides = kForm == kGradW && p.out_fp32 ? 2 : 1;        // 32 columns of fp32 are two store tiles
      for (int side = 0; side < sides; ++side) {
        if (lane == 0) bulk_wait_read_all();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 piece;
          if (sides == 2) {
            // (selected by a loop-invariant condition: v stays in registers)
            piece = side == 0 ? make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3])
                              : make_uint4(v[16 + 4 * q], v[17 + 4 * q], v[18 + 4 * q], v[19 + 4 * q]);
          } else {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float lo = __uint_as_float(v[8 * q + 2 * j]), hi = __uint_as_float(v[8 * q + 2 * j + 1]);
              w[j] = p.fp16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
            }
            piece = make_uint4(w[0], w[1], w[2], w[3]);
          }
          *reinterpret_cast<uint4*>(store + store_piece(lane, q)) = piece;
        }
        const int x = col + side * 16;
        if (rows_here >= 32 || kForm == kGradW) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if constexpr (kForm == kGradW) tma_store_3d(&p.map_out, store, x, row0, g);
            else tma_store_2d(&p.map_out, store, x, c.begin + row0);
            bulk_commit_group();
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = k * 8 + (lane >> 2), piece = lane & 3;
            if (row < rows_here && x + piece * 8 < p.n_total)
              *reinterpret_cast<uint4*>(p.out + static_cast<long long>(c.begin + row0 + row) * p.ld_out + 2 * (x + piece * 8)) =
                  *reinterpret_cast<const uint4*>(store + store_piece(row, piece));
          }
        }
      }
    };
    constexpr int kChunks = kTile / 64;             // chunks of 32 columns of this warp's half
    uint32_t acc = 0;
    for (int t = unit, g = 0; t < total; t += units) {
      const Tile c = tile_at(t, g);
      uint32_t r[kChunks][32];
      if (c.steps == c.first) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) r[i][j] = 0;
      } else {
        const uint32_t as = acc & 1u;
        if (!mbar_wait_warp(&tmem_full_bar[as], (acc >> 1) & 1u, abort_ptr)) { give_up(kStatusRaggedEpilogue); break; }
        ++acc;
        tc_fence_after_sync();
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
          tmem_ld_32x32b_x32(lane_base + as * kTile + half * (kTile / 2) + i * 32, r[i]);
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {                                 // the next tile's MMAs need not wait for the stores
          if constexpr (kPair) mbar_arrive_cluster(mapa_shared(smem_u32(&tmem_empty_bar[as]), 0));
          else mbar_arrive(&tmem_empty_bar[as]);
        }
      }
      if constexpr (kSplit) {
        const bool ok = join_parts(
            smem, &parts_bar, warp - 2, quarter, half, split, part, abort_ptr,
            [&](int j) {
              const uint32_t* q = &r[j >> 3][(j & 7) * 4];
              return make_float4(__uint_as_float(q[0]), __uint_as_float(q[1]), __uint_as_float(q[2]), __uint_as_float(q[3]));
            },
            [&](int row, int col, float4 a, float4 b) {
              row += c.m0;
              col += c.n0;
              if (row >= (kForm == kGradW ? p.m_total : c.count) || col >= p.n_total) return;
              uint8_t* to = p.out + (kForm == kGradW ? g * p.out_group + row * p.ld_out : (c.begin + row) * p.ld_out);
              if (kForm == kGradW && p.out_fp32) {
                reinterpret_cast<float4*>(to + 4 * col)[0] = a;
                reinterpret_cast<float4*>(to + 4 * col)[1] = b;
              } else {
                *reinterpret_cast<uint4*>(to + 2 * col) = pack_8(a, b, p.fp16);
              }
            });
        if (!ok) { give_up(kStatusRaggedEpilogue); break; }
      } else {
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
          emit(c, g, c.m0 + rank * kTileM + quarter * 32, c.n0 + half * (kTile / 2) + i * 32, r[i]);
      }
    }
    if (lane == 0) bulk_wait_all();
    if (kForm != kGradW && p.zero_unused)
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
  if constexpr (kPair || kSplit) cluster_sync_all();      // no CTA leaves while another may still signal it or read from it
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (kPair) tmem_dealloc_pair(tmem_base, kTmemCols);
    else tmem_dealloc(tmem_base, kTmemCols);
  }
}

// 256 x 256 tiles of SM pairs or 128 x 128 tiles of single CTAs.  A step of either takes the same time (the single CTA's is
// bound by shared memory: 32 KB written and 64 KB read for 128 x 128 x 64 products), so what counts for y and d x is how
// many rounds of tiles the SMs go through; as many of either: single CTAs, whose prologue and last tile are shorter.
// Measured (us, pair / single): 4 groups, 2560 -> 6912: 100 rows each, 2 rounds of either, 37.0 / 34.7; 150, 2 and 3:
// 37.9 / 43.5; 500, 4 and 7: 64.3 / 91.4; 6912 -> 2560: 150, 1 and 1: 43.1 / 39.2; 200, 1 and 2: 43.3 / 67.5; 8 groups,
// 2048 -> 2048, 100 rows, 1 and 2: 19.0 / 26.1.  d W, whose contraction is the rows, writes more than it multiplies below
// 256 rows a group: at 200 57.1 / 51.9, 28.9 / 25.7; 300 63.6 / 65.8, 34.4 / 36.3; 900 110.7 / 148.3.  Tiles of 64 columns,
// and pairs with 128, were never the fastest.
static bool pairs_take_fewer_rounds(int64_t rows, int64_t groups, int64_t cols, int sms) {
  return tile_rounds(rows, groups, 2 * kTileM, up_to(cols, 2 * kTileM), 2, sms) <
         tile_rounds(rows, groups, kTileM, up_to(cols, kTileM), 1, sms);
}

// Few tiles with a long contraction are shared by clusters (pick_split).  Measured (us, whole / shared): y at 100 rows,
// 2 groups, 8192 -> 256: 37.6 / 13.5; 2048 -> 512: 13.4 / 10.4; with 16 steps, 1024 -> 256: 9.4 / 9.8; 4 groups,
// 4096 -> 2048, 64 rows: 23.0 / 17.9; dw 512 x 512 of 8000 rows: 41.9 / 18.0.
struct GmmPlan { int ctas, split, tiles; };

static GmmPlan plan_gmm(bool pairs, int64_t tiles, int64_t steps) {
  const int split = pick_split<grouped_matmul_kernel<kGradW, 1, true>>(tiles, steps, 24, kRaggedTailThreads, kGmmTables);
  if (split > 1) return {1, split, static_cast<int>(tiles)};
  return {pairs ? 2 : 1, 1, 0};
}

template <int kForm, int kCtas, bool kSplit>
static int launch_gmm(const GmmParams& p, int cluster, int ctas, cudaStream_t stream) {
  return launch_ragged<grouped_matmul_kernel<kForm, kCtas, kSplit>>(
      p, kForm == kGradW ? kRaggedTailThreads : kRaggedThreads, kGmmTables, cluster, ctas, stream);
}

template <int kForm>
static int launch_gmm_plan(const GmmPlan& plan, GmmParams& p, int sms, cudaStream_t stream) {
  p.split = plan.split;
  if (plan.split > 1) return launch_gmm<kForm, 1, true>(p, plan.split, plan.tiles * plan.split, stream);
  return plan.ctas == 2 ? launch_gmm<kForm, 2, false>(p, 2, sms / 2 * 2, stream) : launch_gmm<kForm, 1, false>(p, 1, sms, stream);
}

static bool rows_ok(const void* p, int64_t ld, int64_t cols, int elem_bytes) {
  return p && aligned16(p) && ld >= cols && ld * elem_bytes % 16 == 0 && cols * elem_bytes % 16 == 0;
}

static int check_gmm(int dtype, int rows, int groups, int n, int k, const int32_t* offsets, const int32_t* status) {
  if (rows < 0 || groups < 0 || n <= 0 || k <= 0 || !status) return COMFY_MOE_EINVAL;
  if (dtype != COMFY_MOE_BF16 && dtype != COMFY_MOE_FP16) return COMFY_MOE_EUNSUPPORTED;
  if (groups > kRaggedMaxGroups || n % 8 || k % 8 || !ragged_sizes_fit(rows, n, k)) return COMFY_MOE_EUNSUPPORTED;
  if (groups > 0 && !offsets) return COMFY_MOE_EINVAL;
  return COMFY_MOE_OK;
}

static uint32_t gmm_idesc(int dtype, int form, int ctas) {
  uint32_t d = umma_idesc<false>(kTileM * ctas, kTileM * ctas);
  if (dtype == COMFY_MOE_FP16) d &= ~((7u << 7) | (7u << 10));       // format 0: both operands fp16
  if (form == kGradW) d |= 1u << 15;                                 // A with its output dimension contiguous
  if (form != kForward) d |= 1u << 16;                               // B with its output dimension contiguous
  return d;
}

}  // namespace comfy_b200

using namespace comfy_b200;

static int rows_by_group(int form, const void* a, int64_t ld_a, const void* w, int64_t ld_w, int64_t w_group_stride,
                         int dtype, int rows, int groups, int n, int k, const int32_t* offsets, const int32_t* counts,
                         int zero_unused, void* out, int64_t ld_out, int32_t* status, void* stream) {
  int rc = check_gmm(dtype, rows, groups, n, k, offsets, status);
  if (rc != COMFY_MOE_OK || rows == 0) return rc;
  const int in = form == kForward ? k : n, cols = form == kForward ? n : k;
  if (!rows_ok(a, ld_a, in, 2) || !rows_ok(out, ld_out, cols, 2)) return COMFY_MOE_EINVAL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (groups == 0) {
    if (zero_unused && cudaMemset2DAsync(out, ld_out * 2, 0, static_cast<size_t>(cols) * 2, rows, s) != cudaSuccess)
      return COMFY_MOE_ECUDA;
    return COMFY_MOE_OK;
  }
  if (!rows_ok(w, ld_w, k, 2) || (groups > 1 && (w_group_stride % 8 || w_group_stride < 0))) return COMFY_MOE_EINVAL;
  const int sms = sm100_count();
  if (sms < 0) return -sms;
  if (form == kForward && rows <= kFewRows) {
    FewParams f;
    memset(&f, 0, sizeof(f));
    f.x = static_cast<const uint8_t*>(a); f.w = static_cast<const uint8_t*>(w); f.out = static_cast<uint8_t*>(out);
    f.offsets = offsets; f.counts = counts;
    f.ld_x = ld_a * 2; f.ld_w = ld_w * 2; f.w_group = w_group_stride * 2; f.ld_out = ld_out * 2;
    f.groups = groups; f.rows = rows; f.n = n; f.k = k; f.zero_unused = zero_unused;
    return launch_few_rows(f, dtype == COMFY_MOE_FP16, s);
  }
  GmmParams p;
  memset(&p, 0, sizeof(p));
  const CUtensorMapDataType t = dtype == COMFY_MOE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const GmmPlan plan = plan_gmm(pairs_take_fewer_rounds(rows, groups, cols, sms),
                                most_row_tiles(rows, groups, kTileM) * up_to(cols, kTileM), up_to(in, kStepK));
  const int ctas = plan.ctas;
  if ((rc = ragged_map(&p.map_a, t, 2, a, in, rows, 0, ld_a, 0, 64, kTileM)) != COMFY_MOE_OK) return rc;
  if ((rc = ragged_map(&p.map_b, t, 2, w, k, n, groups, ld_w, w_group_stride, 64, form == kForward ? kTileM : kStepK)) != COMFY_MOE_OK)
    return rc;
  if ((rc = ragged_map(&p.map_out, t, 2, out, cols, rows, 0, ld_out, 0, 32, 32)) != COMFY_MOE_OK) return rc;
  p.offsets = offsets; p.counts = counts;
  p.out = static_cast<uint8_t*>(out); p.ld_out = ld_out * 2;
  p.status = status;
  p.groups = groups; p.rows = rows;
  p.n_total = cols; p.k_total = in;
  // a band's rows of A stay in L2 (126 MB) beside the panels of W that pass: 32 MB of them
  const int64_t band = (32ll << 20) / (static_cast<int64_t>(kTileM * ctas) * in * 2);
  p.band = static_cast<int>(band < 8 ? 8 : (band > 64 ? 64 : band));
  p.zero_unused = zero_unused;
  p.fp16 = dtype == COMFY_MOE_FP16;
  p.idesc = gmm_idesc(dtype, form, ctas);
  return form == kForward ? launch_gmm_plan<kForward>(plan, p, sms, s) : launch_gmm_plan<kGradX>(plan, p, sms, s);
}

extern "C" int comfy_moe_grouped_matmul(const void* x, int64_t ld_x, const void* w, int64_t ld_w, int64_t w_group_stride,
                                        int dtype, int rows, int n_groups, int out_features, int in_features,
                                        const int32_t* offsets, const int32_t* counts, int zero_unused, void* out,
                                        int64_t ld_out, int32_t* status, void* stream) {
  return rows_by_group(kForward, x, ld_x, w, ld_w, w_group_stride, dtype, rows, n_groups, out_features, in_features, offsets,
                       counts, zero_unused, out, ld_out, status, stream);
}

extern "C" int comfy_moe_grouped_matmul_dgrad(const void* dy, int64_t ld_dy, const void* w, int64_t ld_w,
                                              int64_t w_group_stride, int dtype, int rows, int n_groups, int out_features,
                                              int in_features, const int32_t* offsets, const int32_t* counts,
                                              int zero_unused, void* dx, int64_t ld_dx, int32_t* status, void* stream) {
  return rows_by_group(kGradX, dy, ld_dy, w, ld_w, w_group_stride, dtype, rows, n_groups, out_features, in_features, offsets,
                       counts, zero_unused, dx, ld_dx, status, stream);
}

extern "C" int comfy_moe_grouped_matmul_wgrad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int dtype, int rows,
                                              int n_groups, int out_features, int in_features, const int32_t* offsets,
                                              const int32_t* counts, int out_dtype, void* dw, int64_t ld_dw,
                                              int64_t dw_group_stride, int32_t* status, void* stream) {
  const int n = out_features, k = in_features;
  int rc = check_gmm(dtype, rows, n_groups, n, k, offsets, status);
  if (rc != COMFY_MOE_OK || n_groups == 0) return rc;
  const bool fp32 = out_dtype == COMFY_MOE_FP32;
  if (!fp32 && out_dtype != dtype) return COMFY_MOE_EUNSUPPORTED;
  const int out_bytes = fp32 ? 4 : 2;
  if (!rows_ok(dw, ld_dw, k, out_bytes) || (n_groups > 1 && (dw_group_stride * out_bytes % 16 || dw_group_stride < n * ld_dw)))
    return COMFY_MOE_EINVAL;
  if (rows > 0 && (!rows_ok(dy, ld_dy, n, 2) || !rows_ok(x, ld_x, k, 2))) return COMFY_MOE_EINVAL;
  const int sms = sm100_count();
  if (sms < 0) return -sms;
  GmmParams p;
  memset(&p, 0, sizeof(p));
  const CUtensorMapDataType t = dtype == COMFY_MOE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const int64_t tiles = n_groups * up_to(n, kTileM) * up_to(k, kTileM);
  const GmmPlan plan = plan_gmm(rows >= 256ll * n_groups, tiles, rows / n_groups / kStepK);
  if (rows > 0) {
    if ((rc = ragged_map(&p.map_a, t, 2, dy, n, rows, 0, ld_dy, 0, 64, kStepK)) != COMFY_MOE_OK) return rc;
    if ((rc = ragged_map(&p.map_b, t, 2, x, k, rows, 0, ld_x, 0, 64, kStepK)) != COMFY_MOE_OK) return rc;
  }
  if ((rc = ragged_map(&p.map_out, fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : t, out_bytes, dw, k, n, n_groups, ld_dw,
                       dw_group_stride, fp32 ? 16 : 32, 32)) != COMFY_MOE_OK)
    return rc;
  p.offsets = offsets; p.counts = counts;
  p.out = static_cast<uint8_t*>(dw); p.ld_out = ld_dw * out_bytes; p.out_group = dw_group_stride * out_bytes;
  p.status = status;
  p.groups = n_groups; p.rows = rows;
  p.m_total = n; p.n_total = k;
  p.band = 16;
  p.fp16 = dtype == COMFY_MOE_FP16;
  p.out_fp32 = fp32;
  p.idesc = gmm_idesc(dtype, kGradW, plan.ctas);
  return launch_gmm_plan<kGradW>(plan, p, sms, static_cast<cudaStream_t>(stream));
}
