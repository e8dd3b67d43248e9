// e4m3 with a scale for each block of 128: the rule by which a block is quantised, shared by the quantisers and by the
// products that quantise on the way.  For a block with the largest magnitude m = max(max|x|, 2^-100):
//   scale = m / 448 (fp32),   q = e4m3(x * 448 / m), round to nearest even, as of the exact quotient.
// bf16 and fp16 values have significands of at most 11 bits, and so has m.  A quotient of two such numbers that is no
// border between two e4m3 values (a number of at most 5 significant bits) is at least 2^-16 of itself away from one.  So
// x * (448 / m), two roundings and thus at most two units of 2^-24 off, is rounded to 21 significant bits first: that
// moves a value back onto the border where the quotient is one, and never onto or over one where it is not; the conversion
// then rounds as it would the exact quotient.  A full division per element makes the quantiser bound by instructions
// (17 us for 8192 x 2560 against 12.7).  fp32 values keep the division: ((x * 0.4375) / m) * 1024 has one rounding.
// The floor 2^-100 keeps the scales and their products out of the subnormal range; a block of zeros has zeros.  The maximum is
// taken on the bit patterns, so a NaN or an infinity wins it and reaches every result the block takes part in: its scale
// is then NaN or infinite.
#pragma once
#include <type_traits>

#include "moe_common.cuh"

namespace comfy_b200 {

constexpr uint32_t kTinyBits = (127u - 100u) << 23;                 // 2^-100
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// What a block with the largest magnitude `top` multiplies by, and its scale.
struct BlockScale { float top, inverse; uint32_t half, keep; };
__device__ __forceinline__ BlockScale block_scale(uint32_t top_bits) {
  const float top = __uint_as_float(top_bits);
  const bool finite = top_bits < 0x7f800000u;      // (rounding a NaN's bits would carry into its sign)
  return {top, __fdiv_rn(448.0f, top), finite ? 4u : 0u, finite ? ~7u : ~0u};
}
__device__ __forceinline__ float stored_scale(const BlockScale& s) { return __fdiv_rn(s.top, 448.0f); }
// x * 448 / top, ready for the conversion to e4m3; kShort: x has at most 11 significant bits
template <bool kShort>
__device__ __forceinline__ float block_quotient(const BlockScale& s, float x) {
  if constexpr (kShort) return __uint_as_float((__float_as_uint(x * s.inverse) + s.half) & s.keep);
  else return __fdiv_rn(x * 0.4375f, s.top) * 1024.0f;
}

}  // namespace comfy_b200
