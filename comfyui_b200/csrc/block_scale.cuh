// e4m3 with a scale for each block of 128: the rule by which a block is quantised, shared by the quantisers and by the
// products that quantise on the way.  For a block with the largest magnitude m = max(max|x|, 2^-100):
//   scale = m / 448 (fp32),   q = e4m3(x * 448 / m), round to nearest even, as of the exact quotient.
// A quotient that is no border between two e4m3 values (a number of at most 5 significant bits) keeps away from all of them:
// 448 x / m = 7 X / M times a power of two with whole X and M below 2^p, and a border is B < 2^5 times one, so the two differ
// by at least 1 / (M B) or 1 / (7 X) of themselves, with p = 11 (bf16, fp16) by 2^-16, with p = 24 (fp32) by 2^-29.
// bf16 and fp16: x * (448 / m), two roundings and thus at most two units of 2^-24 off, is rounded to 21 significant bits
// first: that moves a value back onto the border where the quotient is one, and never onto or over one where it is not; the
// conversion then rounds as it would the exact quotient.  A full division per element makes the quantiser bound by
// instructions (17 us for 8192 x 2560 against 12.7).
// fp32: p + e is the quotient to 2^-46 of itself, with p = x * inverse and e what the product and the reciprocal have rounded
// off; s = fl(p + e) lies on the quotient's side of every border that it is not equal to (a border is an fp32 number), and
// what is left, t, tells the side where it is equal: |t| is above 2^-30 of s then, and below 2^-45 where the quotient is the
// border.  So s moves by one unit towards t if t counts and s is even, as borders are: onto no border and over none.
// (8192 x 2560: 22.4 us; ((x * 7 / 16) / m) * 1024, whose product and quotient both round, took 19.4 and missed by a step
// next to borders.)
// The floor 2^-100 keeps a scale normal (2^-109 or more); a block of zeros has zeros.  The product of two scales is taken in
// fp32: it is subnormal, and loses digits, where the two blocks' maxima multiply to less than 2^-108 (results below 2^-101),
// and infinite where they multiply to more than 2^145.  The maximum is taken on the bit patterns, so a NaN or an infinity
// wins it and reaches every result the block takes part in: its scale
// is then NaN or infinite.
#pragma once
#include <type_traits>

#include "moe_common.cuh"

namespace comfy_b200 {

constexpr uint32_t kTinyBits = (127u - 100u) << 23;                 // 2^-100
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// What a block with the largest magnitude `top` multiplies by, and its scale.
struct BlockScale { float top, inverse, low; uint32_t half, keep; };      // low: what inverse lacks, as a share of it
__device__ __forceinline__ BlockScale block_scale(uint32_t top_bits) {
  const float top = __uint_as_float(top_bits);
  const bool finite = top_bits < 0x7f800000u;      // (rounding a NaN's bits would carry into its sign)
  const float inverse = __fdiv_rn(448.0f, top);
  return {top, inverse, finite ? fmaf(-inverse, top, 448.0f) * (1.0f / 448.0f) : 0.f, finite ? 4u : 0u, finite ? ~7u : ~0u};
}
__device__ __forceinline__ float stored_scale(const BlockScale& s) { return __fdiv_rn(s.top, 448.0f); }
// x * 448 / top, ready for the conversion to e4m3; kShort: x has at most 11 significant bits
template <bool kShort>
__device__ __forceinline__ float block_quotient(const BlockScale& s, float x) {
  if constexpr (kShort) {
    return __uint_as_float((__float_as_uint(x * s.inverse) + s.half) & s.keep);
  } else {
    const float p = __fmul_rn(x, s.inverse);
    const float e = fmaf(p, s.low, fmaf(x, s.inverse, -p));
    const float sum = __fadd_rn(p, e), t = __fsub_rn(e, __fsub_rn(sum, p));
    uint32_t bits = __float_as_uint(sum);
    if (fabsf(t) > fabsf(sum) * 0x1p-38f && (bits & 1u) == 0) bits += (t > 0.f) == (sum > 0.f) ? 1u : ~0u;
    return copysignf(__uint_as_float(bits), x);      // (a quotient that underflows keeps its sign)
  }
}

}  // namespace comfy_b200
