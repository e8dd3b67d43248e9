// e4m3 with a scale for each block of 128: the activation quantiser (blocks of 1 x 128 along a row) and the weight
// quantiser (blocks of 128 x 128), by the rule of block_scale.cuh.  Both are bound by HBM: 3 bytes per element of bf16.
#include "block_scale.cuh"

namespace comfy_b200 {

constexpr int kQuantBlock = COMFY_MOE_SCALE_BLOCK;
constexpr int kLaneElems = 16;                        // 16 e4m3 bytes: one store
constexpr int kLanesPerBlock = kQuantBlock / kLaneElems;

template <typename T> struct Lane16 { uint4 raw[sizeof(T)]; };      // 16 elements of T as 16-byte words

template <typename T>
__device__ __forceinline__ void lane_values(const Lane16<T>& in, float (&v)[kLaneElems]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(in.raw);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}

template <bool kShort>
__device__ __forceinline__ uint4 to_e4m3(const float (&v)[kLaneElems], const BlockScale& s) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = block_quotient<kShort>(s, v[4 * i + j]);
    w[i] = static_cast<uint32_t>(f2_to_e4m3x2(q[0], q[1])) | (static_cast<uint32_t>(f2_to_e4m3x2(q[2], q[3])) << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 32 rows x one block per CTA: eight lanes per row, so the maximum needs three shuffles, and the 32 scales of a block are
// one line of the [blocks][rows] scale matrix (what the product's epilogue, one row per lane, reads without gaps).
template <typename T>
__global__ void __launch_bounds__(256)
block_quantize_kernel(const T* __restrict__ x, long long ld, int rows, int cols, uint8_t* __restrict__ q, long long ld_q,
                      float* __restrict__ scale, long long ld_scale) {
  const int row = blockIdx.x * 32 + (threadIdx.x >> 3), l = threadIdx.x & 7;
  const int col = blockIdx.y * kQuantBlock + l * kLaneElems;
  const bool live = row < rows && col < cols;         // cols is a multiple of 16: a lane has all of its elements or none
  Lane16<T> in = {};
  if (live) {
    const uint4* src = reinterpret_cast<const uint4*>(x + row * ld + col);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) in.raw[i] = __ldg(src + i);
  }
  float v[kLaneElems];
  lane_values<T>(in, v);
  uint32_t top = kTinyBits;
#pragma unroll
  for (int i = 0; i < kLaneElems; ++i) top = max(top, magnitude_bits(v[i]));
#pragma unroll
  for (int d = 1; d < kLanesPerBlock; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  const BlockScale s = block_scale(top);
  if (live) *reinterpret_cast<uint4*>(q + row * ld_q + col) = to_e4m3<sizeof(T) == 2>(v, s);
  if (l == 0 && row < rows) scale[blockIdx.y * ld_scale + row] = stored_scale(s);
}

// One 128 x 128 block per CTA, held in registers between the maximum and the division.
template <typename T>
__global__ void __launch_bounds__(256)
block_quantize_weight_kernel(const T* __restrict__ w, long long ld, long long group_stride, int n, int k,
                             uint8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t s_top[8];
  const int l = threadIdx.x & 7, r0 = threadIdx.x >> 3;
  const int col = blockIdx.x * kQuantBlock + l * kLaneElems;
  const T* src = w + blockIdx.z * group_stride;
  Lane16<T> in[4] = {};
  uint32_t top = kTinyBits;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = blockIdx.y * kQuantBlock + i * 32 + r0;
    if (row < n && col < k) {
      const uint4* p = reinterpret_cast<const uint4*>(src + row * ld + col);
#pragma unroll
      for (int j = 0; j < static_cast<int>(sizeof(T)); ++j) in[i].raw[j] = __ldg(p + j);
    }
    float v[kLaneElems];
    lane_values<T>(in[i], v);
#pragma unroll
    for (int j = 0; j < kLaneElems; ++j) top = max(top, magnitude_bits(v[j]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, s_top[i]);
  const BlockScale s = block_scale(top);
  if (threadIdx.x == 0) scale[(static_cast<long long>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = stored_scale(s);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = blockIdx.y * kQuantBlock + i * 32 + r0;
    if (row < n && col < k) {
      float v[kLaneElems];
      lane_values<T>(in[i], v);
      *reinterpret_cast<uint4*>(q + (static_cast<long long>(blockIdx.z) * n + row) * k + col) = to_e4m3<sizeof(T) == 2>(v, s);
    }
  }
}

static int elem_bytes(int dtype) {
  return dtype == COMFY_MOE_BF16 || dtype == COMFY_MOE_FP16 ? 2 : (dtype == COMFY_MOE_FP32 ? 4 : 0);
}

}  // namespace comfy_b200

using namespace comfy_b200;

extern "C" int comfy_moe_block_quantize(const void* x, int64_t ld_x, int dtype, int rows, int cols, void* out, int64_t ld_out,
                                        float* scale, int64_t ld_scale, void* stream) {
  const int bytes = elem_bytes(dtype);
  if (!bytes || cols % 16 || rows > COMFY_MOE_RAGGED_MAX_ROWS || cols > COMFY_MOE_MAX_SCALE_BLOCKS * kQuantBlock)
    return COMFY_MOE_EUNSUPPORTED;
  if (rows < 0 || cols <= 0) return COMFY_MOE_EINVAL;
  if (rows == 0) return COMFY_MOE_OK;
  if (!x || !out || !scale || !aligned16(x) || !aligned16(out) || ld_x < cols || ld_x * bytes % 16 || ld_out < cols ||
      ld_out % 16 || ld_scale < rows)
    return COMFY_MOE_EINVAL;
  const dim3 grid((rows + 31) / 32, (cols + kQuantBlock - 1) / kQuantBlock);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* q = static_cast<uint8_t*>(out);
  if (dtype == COMFY_MOE_BF16)
    block_quantize_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(x), ld_x, rows, cols, q, ld_out, scale, ld_scale);
  else if (dtype == COMFY_MOE_FP16)
    block_quantize_kernel<__half><<<grid, 256, 0, s>>>(static_cast<const __half*>(x), ld_x, rows, cols, q, ld_out, scale, ld_scale);
  else
    block_quantize_kernel<float><<<grid, 256, 0, s>>>(static_cast<const float*>(x), ld_x, rows, cols, q, ld_out, scale, ld_scale);
  return check_launch();
}

extern "C" int comfy_moe_block_quantize_weight(const void* w, int64_t ld_w, int64_t w_group_stride, int dtype, int n_groups,
                                               int out_features, int in_features, void* out, float* scale, void* stream) {
  const int bytes = elem_bytes(dtype), n = out_features, k = in_features;
  constexpr int kMost = COMFY_MOE_MAX_SCALE_BLOCKS * kQuantBlock;
  if (!bytes || k % 16 || k > kMost || n > kMost || n_groups > COMFY_MOE_MAX_SCALE_BLOCKS) return COMFY_MOE_EUNSUPPORTED;
  if (n_groups < 0 || n <= 0 || k <= 0) return COMFY_MOE_EINVAL;
  if (n_groups == 0) return COMFY_MOE_OK;
  if (!w || !out || !scale || !aligned16(w) || !aligned16(out) || ld_w < k || ld_w * bytes % 16 ||
      (n_groups > 1 && w_group_stride * bytes % 16))
    return COMFY_MOE_EINVAL;
  const dim3 grid((k + kQuantBlock - 1) / kQuantBlock, (n + kQuantBlock - 1) / kQuantBlock, n_groups);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* q = static_cast<uint8_t*>(out);
  if (dtype == COMFY_MOE_BF16)
    block_quantize_weight_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(w), ld_w, w_group_stride, n, k, q, scale);
  else if (dtype == COMFY_MOE_FP16)
    block_quantize_weight_kernel<__half><<<grid, 256, 0, s>>>(static_cast<const __half*>(w), ld_w, w_group_stride, n, k, q, scale);
  else
    block_quantize_weight_kernel<float><<<grid, 256, 0, s>>>(static_cast<const float*>(w), ld_w, w_group_stride, n, k, q, scale);
  return check_launch();
}
