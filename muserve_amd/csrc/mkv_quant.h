// mkv_quant.h — the quantisers of the fp8 and the 4-bit pools, shared by their
// appends and by the append that norms and rotates on the way.
#pragma once

#include "mkv_device.h"

namespace mkv {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float bf16_lo(uint32_t w) { return bits_f32(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return bits_f32(w & 0xffff0000u); }

// torch.clamp(x, -448, 448): NaN passes through unchanged.
__device__ __forceinline__ float clamp448(float x) {
  return x < -448.0f ? -448.0f : (x > 448.0f ? 448.0f : x);
}

// fp8: quantises one row held as N bf16 values (N / 2 words) per lane of a
// LANES-lane group: the lane's N codes, and the row's scale in every lane.
template <int LANES, int N>
__device__ __forceinline__ float quantise_fp8(const uint32_t (&w)[N / 2], uint32_t (&codes)[N / 4]) {
  float x[N];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    x[2 * i] = bf16_lo(w[i]);
    x[2 * i + 1] = bf16_hi(w[i]);
  }
  // absmax over the row. On |x| bit patterns integer max is float max, and
  // any NaN (above +inf as an integer) wins, as torch's amax propagates NaN.
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t ab = f32_bits(x[i]) & 0x7fffffffu;
    m = ab > m ? ab : m;
  }
#pragma unroll
  for (int off = LANES / 2; off >= 1; off >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, off, LANES);
    m = o > m ? o : m;
  }
  const float amax = bits_f32(m);
  const float clamped = amax < 1e-12f ? 1e-12f : amax;  // .clamp(min=1e-12); NaN stays
  const float scale = clamped / 448.0f;
  const float recip = 1.0f / scale;
  float q[N];
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = clamp448(div_by_recip(x[i], scale, recip));
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
    codes[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], lo, true);
  }
  return scale;
}

// ---- 4 bits: e2m1 codes with one power of two for every 32 dims -------------------
//
// A row of a (token, head) of 256 dims is kFp4Row bytes: 128 bytes of codes (the even
// dim in a byte's low half), then the 8 blocks' scales as e8m0 bytes (2^(byte - 127)).
// One contiguous row: a page's 16 rows are 17 lines of 128 bytes, read and written
// whole; scales in a plane of their own would be one more place in HBM for each page.
constexpr int kFp4Block = 32;
constexpr int kFp4Codes = 128;
constexpr int kFp4Row = kFp4Codes + 256 / kFp4Block;
constexpr uint32_t kFp4Nan = 255;  // a block that held an inf or a NaN: reads back as NaN

// The scale byte of a block whose largest |x| has the bf16 bits m: the least power of
// two 2^e with |x| <= 7 * 2^e (e2m1 ends at 6, and what lies between 6 and 7 is nearest
// to 6; on normal values this has the least squared error of the thresholds between 6
// and 8: 0.0125 of the variance, 0.0133 and 0.0132 at these two). e is kept in
// [-120, 125], so that every value, and every half of a code's step, is a normal finite
// bf16 (larger values are held as 6 * 2^125, smaller ones than 2^-122 as 0).
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t m) {
  if (m >= 0x7f80u) return kFp4Nan;
  const int b = (int)((m + 0x1fu) >> 7) - 2;  // (a mantissa above 1.75 carries)
  return (uint32_t)(b < 7 ? 7 : (b > 252 ? 252 : b));
}

// A scale byte as the conversions take it: they go by the exponent bits alone, and
// give NaN for all of them set.
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return bits_f32(byte << 23); }

// Quantises N bf16 values a lane; 32 / N neighbouring lanes hold a block. The lane's N
// codes, and its block's scale byte in each of those lanes. x / 2^e is exact and the
// conversion rounds to nearest even, saturating at 6.
template <int N>
__device__ __forceinline__ uint32_t quantise_fp4(const uint32_t (&w)[N / 2], uint32_t (&codes)[N / 8]) {
  static_assert(N == 8 || N == 16, "4 or 2 lanes a block");
  uint32_t m = 0;  // on |x|'s bits integer max is float max
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
    m = m > lo ? m : lo;
    m = m > hi ? m : hi;
  }
  m = over_lanes<kFp4Block / N>(m, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  const uint32_t byte = fp4_scale_byte(m);
  const float scale = fp4_scale(byte);
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[4 * i]), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[4 * i + 1]), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[4 * i + 2]), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[4 * i + 3]), scale, 3);
    codes[i] = byte == kFp4Nan ? 0u : c;
  }
  return byte;
}

// Codes 2 * PAIR, 2 * PAIR + 1 of a word of 8, times the scale, as a bf16 pair: exact
// (a code has two significant bits). A macro: the byte is an immediate.
#define mkv_fp4_pair(word, pair, scale)                                                    \
  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((word), (scale), (pair)))

}  // namespace mkv
