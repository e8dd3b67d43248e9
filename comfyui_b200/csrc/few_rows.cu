// Products of a few rows with weights that are read once: the single-token form of the grouped products and of the
// block-scaled ones.  At up to 16 rows the weights are all there is to move (2 flops per byte and row), so the work is cut
// for HBM: a block takes 16 output columns of one group over the whole contraction, its eight warps the chunks of it in
// turns, and every lane asks for ten 16-byte pieces of weights before it uses the first.  The arithmetic is one mma.sync tile
// per eight rows: 16 output columns x 8 rows, A = weights, B = rows, both operands in the registers that the loads filled: the
// tile's steps of the contraction may come in any order as long as both sides agree, so a lane's 16 contiguous bytes serve
// two MMAs without a shuffle or shared memory.  (tcgen05 would need both operands in shared memory and 128 rows of one of
// them.)  The warps' partial sums are joined in a fixed order: the result is the same every time.
// Measured (device time, us, cold weights, against the tcgen05 kernels): bf16 2560 -> 6912, one group, 1 row 8.1 / 18.5, 16
// rows 10.6 / 17.7 (HBM: 5.4); four groups, 8 rows 24.0 / 43.2 (all of them busy: 21.6); eight groups 2048 -> 8192, 16 rows
// 53 / 64 (41).
// How many of the ten loads are in flight is the compiler's choice of registers.  Four blocks to an SM leave it 64 and are the
// best of what was measured: with 40, its own choice, it takes them in turns (1 row 10.3, 16 rows 13.3, four groups 25.2, eight
// 63); five blocks of 48: 8.7, 12.6, 26, 59; three of 80: 8.4, 9.4, 28, 57; two of 96: 11.0, 13.0, 32, 63.
#include "block_scale.cuh"
#include "few_rows.cuh"
#include "ragged.cuh"

namespace comfy_b200 {

constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewCols = 16;                   // output columns per block
constexpr int kFewBlocks = 4;                  // of the unscaled kernel, to an SM

// No more groups than rows have any: a grid has that many of them, few_slots.  Blocks (., slot) take group `slot` where
// that is every group, else the slot-th group that has rows; false: there is none for them.  The same in every lane of a warp.
// (With blocks for every group, busy or not: bf16 1024 -> 2048, 8 rows in 8 of 768 groups 208 us, now 20; of 64 groups 20, now
// 10; block-scaled 2560 -> 6912, 2 rows in 2 of 4 groups 14.8, now 13.5.)
__host__ __device__ __forceinline__ int few_slots(const FewParams& p) { return p.groups < p.rows ? p.groups : p.rows; }

// kSeek: groups > rows.  (A variant of its own: with both ways in one kernel 8 block-scaled rows in four groups, 2560 -> 6912,
// took 23.6 us against 22.2.)
template <bool kSeek>
__device__ __forceinline__ bool few_group(const FewParams& p, int slot, int& group, int& begin, int& count) {
  const int lane = threadIdx.x & 31;
  count = 0;
  if constexpr (!kSeek) {
    group = slot;
    if (!p.offsets) {
      begin = 0;
      count = p.rows;
    } else {
      int reach = 0;
      for (int i = lane; i <= slot; i += 32) reach = max(reach, min(max(p.offsets[i], 0), p.rows));
      begin = __reduce_max_sync(0xffffffffu, reach);
      count = max(begin, min(max(p.offsets[slot + 1], 0), p.rows)) - begin;
    }
    if (p.counts) count = min(count, max(p.counts[slot], 0));
  } else {
    int reach = 0, seen = 0;
#pragma unroll 4
    for (int g0 = 0; g0 < p.groups; g0 += 32) {       // (to the end: without a way out the loads go ahead)
      int lo, n;
      ragged_chunk(p.offsets, p.counts, p.groups, p.rows, g0 + lane, reach, lo, n);
      const uint32_t busy = __ballot_sync(0xffffffffu, n > 0);
      const uint32_t mine = __ballot_sync(0xffffffffu, n > 0 && seen + __popc(busy & ((1u << lane) - 1)) == slot);
      if (mine) {
        const int from = __ffs(mine) - 1;
        group = g0 + from;
        begin = __shfl_sync(0xffffffffu, lo, from);
        count = __shfl_sync(0xffffffffu, n, from);
      }
      seen += __popc(busy);
    }
  }
  return count > 0;
}

__device__ __forceinline__ uint4 load_once(const void* p) {     // streamed: read by this block only
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint2 load_row(const void* p) {      // (volatile: behind the loads of weights that precede it)
  uint2 v;
  asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16x8x32_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Joins the warps' 16 x 8 kTiles sums (in the order of the warps) and writes rows [row0, row0 + live) of the result.
template <typename T, int kTiles>
__device__ __forceinline__ void few_store(const FewParams& p, float (&part)[kFewWarps][kFewCols][8 * kTiles + 1],
                                          const float (&c)[kTiles][4], int row0, int live, int n0) {
  const int warp = threadIdx.x >> 5, g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
  for (int j = 0; j < kTiles; ++j) {
    part[warp][g][j * 8 + 2 * t] = c[j][0];
    part[warp][g][j * 8 + 2 * t + 1] = c[j][1];
    part[warp][g + 8][j * 8 + 2 * t] = c[j][2];
    part[warp][g + 8][j * 8 + 2 * t + 1] = c[j][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kFewCols * 8 * kTiles; i += kFewThreads) {
    const int col = i % kFewCols, row = i / kFewCols;
    if (row >= live || n0 + col >= p.n) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) sum += part[w][col][row];
    if (p.bias) sum += to_float(static_cast<const T*>(p.bias)[n0 + col]);
    reinterpret_cast<T*>(p.out + static_cast<long long>(row0 + row) * p.ld_out)[n0 + col] = from_float<T>(sum);
  }
}

// Block (0, few_slots): the rows of no group; there are few enough for one bit each.
__device__ __forceinline__ void few_zero(const FewParams& p) {
  if (blockIdx.x != 0) return;
  const int lane = threadIdx.x & 31;
  uint32_t used = 0;
  int reach = 0;
#pragma unroll 4
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    int lo, n;
    ragged_chunk(p.offsets, p.counts, p.groups, p.rows, g0 + lane, reach, lo, n);
    used |= ((1u << n) - 1) << lo;
  }
  used = __reduce_or_sync(0xffffffffu, used);
  for (int row = threadIdx.x >> 5; row < p.rows; row += kFewWarps)
    if ((used >> row & 1) == 0)
      for (int b = lane * 16; b < 2 * p.n; b += 512)
        *reinterpret_cast<uint4*>(p.out + static_cast<long long>(row) * p.ld_out + b) = make_uint4(0, 0, 0, 0);
}

template <typename T, int kTiles, bool kSeek>
__global__ void __launch_bounds__(kFewThreads, kFewBlocks) few_rows_kernel(const FewParams p) {
  __shared__ float part[kFewWarps][kFewCols][8 * kTiles + 1];
  if (blockIdx.y == few_slots(p)) { few_zero(p); return; }
  int grp, begin, count;
  if (!few_group<kSeek>(p, blockIdx.y, grp, begin, count)) return;
  const int warp = threadIdx.x >> 5, g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
  const int n0 = blockIdx.x * kFewCols;
  const uint8_t* w0 = p.w + grp * p.w_group + static_cast<long long>(n0 + g) * p.ld_w;
  const bool col0 = n0 + g < p.n, col1 = n0 + g + 8 < p.n;
  constexpr int kChunk = 32;                   // elements of the contraction per warp and turn: 64 bytes of a row
  constexpr int kFlight = 5;                   // turns whose loads are in flight together
  const int chunks = (p.k + kChunk - 1) / kChunk;
  float c[kTiles][4] = {};
  for (int i0 = warp; i0 < chunks; i0 += kFewWarps * kFlight) {
    uint4 w[kFlight][2], x[kFlight][kTiles];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int k0 = (i0 + i * kFewWarps) * kChunk + t * 8;            // K is a multiple of 8: a lane has all 8 or none
      const bool in = k0 < p.k;
      w[i][0] = in && col0 ? load_once(w0 + 2 * k0) : make_uint4(0, 0, 0, 0);
      w[i][1] = in && col1 ? load_once(w0 + 8 * p.ld_w + 2 * k0) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        const int row = j * 8 + g;
        x[i][j] = in && row < count ? __ldg(reinterpret_cast<const uint4*>(p.x + static_cast<long long>(begin + row) * p.ld_x + 2 * k0))
                                    : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i)
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        mma_16x8x16<T>(c[j], w[i][0].x, w[i][1].x, w[i][0].y, w[i][1].y, x[i][j].x, x[i][j].y);
        mma_16x8x16<T>(c[j], w[i][0].z, w[i][1].z, w[i][0].w, w[i][1].w, x[i][j].z, x[i][j].w);
      }
  }
  few_store<T, kTiles>(p, part, c, begin, count, n0);
}

// Block-scaled.  kQuantise: one or two rows are quantised here, by every block again (by the rule of block_scale.cuh; each
// warp the blocks that it multiplies), while its weights are on their way: no workspace, one launch.  That costs 1.2 us a
// row at 2560 -> 6912, a launch of the quantiser 1.7 us and the host 3 us, so from three rows on, up to eight, they come
// quantised.  Measured as above: one group, 1 row 8.3 / 12.7, 8 rows 8.3 / 12.7 (HBM: 2.7); four groups, 8 rows 22.2 / 30.3;
// 1024 -> 1024, 8 rows 4.9 / 8.5.  (16 rows, two tiles: 12.1 / 12.4, four groups 28.1 / 30.4, eight 50 / 40: left to tcgen05.)
constexpr int kFewBlk = COMFY_MOE_SCALE_BLOCK;

template <typename T, bool kQuantise, bool kSeek>
__global__ void __launch_bounds__(kFewThreads) few_rows_block_kernel(const FewParams p) {
  extern __shared__ __align__(16) uint8_t xq[];            // kQuantise: [blocks of the contraction][rows][128]
  __shared__ float part[kFewWarps][kFewCols][9];
  if (blockIdx.y == few_slots(p)) { few_zero(p); return; }
  int grp, begin, count;
  if (!few_group<kSeek>(p, blockIdx.y, grp, begin, count)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kFewCols;
  const uint8_t* w0 = p.w + grp * p.w_group + static_cast<long long>(n0 + g) * p.ld_w;
  const bool col0 = n0 + g < p.n, col1 = n0 + g + 8 < p.n;
  const int blocks = (p.k + kFewBlk - 1) / kFewBlk;
  const float* ws = p.ws + grp * p.ws_group + static_cast<long long>(n0 / kFewBlk) * blocks;
  constexpr int kFlight = 3;                   // blocks whose weights are in flight together
  float sum[1][4] = {};
  for (int b0 = warp; b0 < blocks; b0 += kFewWarps * kFlight) {
    uint4 w[kFlight][2][2];
    float scale[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int b = b0 + i * kFewWarps;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k0 = b * kFewBlk + s * 64 + t * 16;                    // K is a multiple of 16
        const bool in = b < blocks && k0 < p.k;
        w[i][s][0] = in && col0 ? load_once(w0 + k0) : make_uint4(0, 0, 0, 0);
        w[i][s][1] = in && col1 ? load_once(w0 + 8 * p.ld_w + k0) : make_uint4(0, 0, 0, 0);
      }
      scale[i] = b < blocks ? __ldg(ws + b) : 0.f;
    }
    float xs[kFlight][2] = {};                 // scales of rows 2 t and 2 t + 1, this lane's columns of the product
    if constexpr (kQuantise) {
      for (int row = 0; row < count; ++row) {
        const uint8_t* src = p.x + static_cast<long long>(begin + row) * p.ld_x;
        uint2 raw[kFlight];
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          const int k0 = (b0 + i * kFewWarps) * kFewBlk + lane * 4;
          raw[i] = k0 < p.k ? load_row(src + 2 * k0) : make_uint2(0, 0);
        }
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          const T* e = reinterpret_cast<const T*>(&raw[i]);
          float v[4];
          uint32_t top = kTinyBits;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            v[q] = to_float(e[q]);
            top = max(top, magnitude_bits(v[q]));
          }
          top = __reduce_max_sync(0xffffffffu, top);
          const BlockScale bs = block_scale(top);
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = block_quotient<true>(bs, v[q]);
          if (b0 + i * kFewWarps < blocks)
            reinterpret_cast<uint32_t*>(xq + ((b0 + i * kFewWarps) * kFewRowsQuantise + row) * kFewBlk)[lane] =
                static_cast<uint32_t>(f2_to_e4m3x2(v[0], v[1])) | (static_cast<uint32_t>(f2_to_e4m3x2(v[2], v[3])) << 16);
          const float s = stored_scale(bs);
          if (row == 2 * t) xs[i][0] = s;
          if (row == 2 * t + 1) xs[i][1] = s;
        }
      }
      __syncwarp();
    } else {
#pragma unroll
      for (int i = 0; i < kFlight; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int b = b0 + i * kFewWarps, row = 2 * t + h;
          if (b < blocks && row < count) xs[i][h] = __ldg(p.xs + b * p.ld_xs + begin + row);
        }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int b = b0 + i * kFewWarps;
      float c[4] = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k0 = b * kFewBlk + s * 64 + t * 16;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (g < count && k0 < p.k) {
          if constexpr (kQuantise)
            x = *reinterpret_cast<const uint4*>(xq + (b * kFewRowsQuantise + g) * kFewBlk + s * 64 + t * 16);
          else
            x = __ldg(reinterpret_cast<const uint4*>(p.x + static_cast<long long>(begin + g) * p.ld_x + k0));
        }
        mma_16x8x32_e4m3(c, w[i][s][0].x, w[i][s][1].x, w[i][s][0].y, w[i][s][1].y, x.x, x.y);
        mma_16x8x32_e4m3(c, w[i][s][0].z, w[i][s][1].z, w[i][s][0].w, w[i][s][1].w, x.z, x.w);
      }
      // (a row or a block that is not there has zeros and the scale 0)
      sum[0][0] = fmaf(c[0], xs[i][0] * scale[i], sum[0][0]);
      sum[0][1] = fmaf(c[1], xs[i][1] * scale[i], sum[0][1]);
      sum[0][2] = fmaf(c[2], xs[i][0] * scale[i], sum[0][2]);
      sum[0][3] = fmaf(c[3], xs[i][1] * scale[i], sum[0][3]);
    }
  }
  few_store<T, 1>(p, part, sum, begin, count, n0);
}

template <auto kKernel>
static int launch_few(const FewParams& p, size_t smem, size_t most, cudaStream_t stream) {
  // one slot more for rows of no group: without offsets the one group has all rows, unless counts say fewer
  const dim3 grid((p.n + kFewCols - 1) / kFewCols, few_slots(p) + (p.zero_unused && (p.offsets || p.counts) ? 1 : 0));
  if (smem > 32 * 1024) {                      // beyond what a kernel may have unasked, beside its static part
    const int rc = allow_shared_memory<kKernel>(most);
    if (rc != COMFY_MOE_OK) return rc;
  }
  kKernel<<<grid, kFewThreads, smem, stream>>>(p);
  return check_launch();
}

template <typename T, bool kSeek>
static int launch_rows_typed(const FewParams& p, cudaStream_t stream) {
  return p.rows <= 8 ? launch_few<few_rows_kernel<T, 1, kSeek>>(p, 0, 0, stream)
                     : launch_few<few_rows_kernel<T, 2, kSeek>>(p, 0, 0, stream);
}

int launch_few_rows(const FewParams& p, bool fp16, cudaStream_t stream) {
  if (p.groups > p.rows)
    return fp16 ? launch_rows_typed<__half, true>(p, stream) : launch_rows_typed<__nv_bfloat16, true>(p, stream);
  return fp16 ? launch_rows_typed<__half, false>(p, stream) : launch_rows_typed<__nv_bfloat16, false>(p, stream);
}

template <typename T, bool kSeek>
static int launch_block_typed(const FewParams& p, cudaStream_t stream) {
  if (p.xs == nullptr)
    return launch_few<few_rows_block_kernel<T, true, kSeek>>(
        p, static_cast<size_t>((p.k + kFewBlk - 1) / kFewBlk) * kFewRowsQuantise * kFewBlk,
        static_cast<size_t>(kFewQuantiseMaxK) * kFewRowsQuantise, stream);
  return launch_few<few_rows_block_kernel<T, false, kSeek>>(p, 0, 0, stream);
}

int launch_few_rows_block(const FewParams& p, bool fp16, cudaStream_t stream) {
  if (p.groups > p.rows)
    return fp16 ? launch_block_typed<__half, true>(p, stream) : launch_block_typed<__nv_bfloat16, true>(p, stream);
  return fp16 ? launch_block_typed<__half, false>(p, stream) : launch_block_typed<__nv_bfloat16, false>(p, stream);
}

}  // namespace comfy_b200
