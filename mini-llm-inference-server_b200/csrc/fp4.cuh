// The 4-bit pool format and its conversions.
//
// A pool is uint8 [num_blocks][Hkv][17][Dh / 2]: one contiguous record per (block, head), so a page of one head
// is a single run of 8.5 Dh bytes (1088 for Dh 128; 0.266 of the 16-bit page).  Rows 0..15 are the tokens' codes,
// two e2m1 values a byte (dim 2i in the low nibble).  Row 16 holds the scales, one byte for each run of 32 dims
// of a token, at [run][2 * (token % 8) + token / 8]: the byte of token g next to token g + 8's, the pair of rows
// that one thread of a tensor-core fragment holds.  A scale byte b stands for the fp16 with bits b << 7 (5
// exponent and 3 mantissa bits, no sign), so widening it is a shift.
// value = code * scale: e2m1 has 2 significant bits and the scale 4, so a value has at most 6 and is exact in
// bf16 and fp16 (6 * the largest scale, 61440, is a finite fp16; the smallest step, 2^-18, an fp16 subnormal).
#pragma once

#include "common.cuh"

namespace mlb {

constexpr int kFp4Run = 32;                // dims that share a scale
constexpr float kFp4TopValue = 61440.f;    // 6 * the largest scale (10240): larger magnitudes are stored as this
constexpr int kFp4Rows = kBlockSize + 1;   // 16 rows of codes, one of scales

template <int DH>
struct Fp4 {
  static constexpr int kRow = DH / 2;                    // bytes of one token's codes
  static constexpr int kScales = kBlockSize * kRow;      // offset of the scale row
  static constexpr int kRecord = kFp4Rows * kRow;        // one (block, head)
  static_assert(kRecord % 16 == 0, "records start 16-byte aligned");
};

// offset of a scale byte in the scale row
__host__ __device__ constexpr int fp4_scale_at(int run, int token) { return run * kBlockSize + 2 * (token & 7) + (token >> 3); }

// 8 codes (one 32-bit word) -> 4 pairs of fp16, dims in order
__device__ __forceinline__ void fp4_unpack8(uint32_t w, uint32_t& h0, uint32_t& h1, uint32_t& h2, uint32_t& h3) {
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}\n"
      : "=r"(h0), "=r"(h1), "=r"(h2), "=r"(h3)
      : "r"(w));
}

__device__ __forceinline__ uint32_t hmul2_u32(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// 8 values -> one word of codes; nearest level, ties to even codes (cvt), sign kept
__device__ __forceinline__ uint32_t fp4_pack8(const float (&r)[8]) {
  uint32_t w;
  asm("{\n.reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n}\n"
      : "=r"(w)
      : "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]));
  return w;
}

// y = amax / 6 (exact, or cut towards zero with its last bit set) -> the nearest scale byte, ties to even.
__device__ __forceinline__ uint32_t fp4_round_scale(float y) {
  if (y < 6.103515625e-05f) return static_cast<uint32_t>(__float2uint_rn(y * 131072.f));  // below 2^-14: steps of 2^-17
  uint32_t u = __float_as_uint(y);
  u += 0x7ffffu + ((u >> 20) & 1u);       // to 3 mantissa bits, nearest even
  return (u >> 20) - ((127u - 15u) << 3);  // exponent bias 15
}

// Scale byte of a run whose largest magnitude is amax (at most kFp4TopValue).  fp32: the quotient is cut towards zero
// and its last bit set when anything was cut off, so the rounding to the byte sees which side of a tie the true
// quotient lies on.
__device__ __forceinline__ uint32_t fp4_scale_byte(float amax) {
  float y = __fdiv_rz(amax, 6.f);
  if (fmaf(-y, 6.f, amax) != 0.f) y = __uint_as_float(__float_as_uint(y) | 1u);
  return fp4_round_scale(y);
}
// The same for an amax of at most 11 significant bits: a product with 1/6 is exact where amax / 6 is a tie (5 bits; all
// 16 mantissas checked), and elsewhere the quotient lies 2^-11 or more from a tie.
__device__ __forceinline__ uint32_t fp4_scale_byte_16(float amax) { return fp4_round_scale(amax * (1.f / 6.f)); }

__device__ __forceinline__ float fp4_scale_value(uint32_t byte) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(byte << 7)));
}

// 1 / scale as hi + lo, hi at most the true reciprocal (the approximation, within a unit, less one unit) and lo >= 0,
// together good to 2^-46; zeros for a zero scale.  x * hi + x * lo in one rounding is then exact where x / scale is a
// border between two levels, keeps the sign of a zero, and for x of at most 11 significant bits crosses no border.
__device__ __forceinline__ void fp4_reciprocal(float scale, float& hi, float& lo) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
  hi = scale > 0.f ? __uint_as_float(__float_as_uint(r) - 1u) : 0.f;
  lo = scale > 0.f ? fmaf(-hi, scale, 1.f) * hi : 0.f;
}
// x: of at most 11 significant bits; two quotients by packed operations.
__device__ __forceinline__ void fp4_quotients_16(float& x0, float& x1, float hi, float lo) {
  asm("{\n.reg .b64 x, h, l;\nmov.b64 x, {%0, %1};\nmov.b64 h, {%2, %2};\nmov.b64 l, {%3, %3};\n"
      "mul.rn.f32x2 l, x, l;\nfma.rn.f32x2 x, x, h, l;\nmov.b64 {%0, %1}, x;\n}\n"
      : "+f"(x0), "+f"(x1)
      : "f"(hi), "f"(lo));
}

// The same for fp32 x, whose quotients can round onto a border that they only lie next to: an inexact quotient is made
// odd in the direction of its remainder.
__device__ __forceinline__ float fp4_quotient_32(float x, float scale, float hi, float lo) {
  const float q = fmaf(x, hi, x * lo);
  const float r = fmaf(-q, scale, x);
  uint32_t u = __float_as_uint(q);
  if (r != 0.f && !(u & 1u) && (u << 1) != 0u) u += ((__float_as_uint(r) ^ u) >> 31) ? 0xffffffffu : 1u;
  return __uint_as_float(u);
}

// P in fp16.  A row's probabilities are 2^(score - m) with m between kFp4Lift and kFp4Lift + kFp4Rise below the largest
// score so far: at most 2^14, and normal fp16 numbers (2^-11 relative) down to 2^-24 of the largest one.  Below that they
// lie on a grid of 2^-34 of it (with m at the largest score itself the grid is 2^-24, and the weight of 40000 keys that
// e^18 divides, a thousandth of the row, was lost).  m moves when a score rises by more than kFp4Rise above the one it was
// taken from, which after the first pages is rare; sums and O are fp32 and carry the lift until O is divided by the sum.
constexpr float kFp4Lift = 10.f;
constexpr float kFp4Rise = 4.f;

// bf16 query rows enter fp16 products divided by a power of two that brings their largest element mx to [2^14, 2^15):
// down = 2^-e, up = 2^e, both normal numbers (a row below 2^-112 stays below 2^14).  A bf16 element keeps its 8 bits
// down to 2^-31 of the row's largest (the lowest of them then weighs 2^-24, the step of fp16's subnormal numbers), and
// smaller ones lie on a grid of 2^-38 of it: finer than what an fp32 sum with the row's largest would leave of them.
// Sums stay far inside fp32: 2^15 x 61440 x 256 products is below 2^39.
__device__ __forceinline__ void fp4_query_scale(float mx, float& up, float& down) {
  const int e = max(1, static_cast<int>(__float_as_uint(mx) >> 23) - 14);  // biased exponent, at most 241
  down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
  up = __uint_as_float(static_cast<uint32_t>(e) << 23);
}
// The softmax scale of such a row: a positive finite number.  At zero a masked score (-inf) would become NaN; at or
// below the smallest normal number every weight is 1 (sums of products stay below 2^39, so exponents below 2^-87).
__device__ __forceinline__ float fp4_softmax_scale(float sl2, float up) {
  return fminf(fmaxf(sl2 * up, 1.17549435e-38f), 3.4028235e38f);
}

}  // namespace mlb
