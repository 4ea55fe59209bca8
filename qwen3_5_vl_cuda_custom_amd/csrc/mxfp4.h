// Microscaled 4-bit floating point (MXFP4) on gfx950.
//
// A row is cut into blocks of 32 consecutive values. A value is a 4-bit float
// (E2M1: sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6), a block has one power-of-two
// scale held as its exponent (E8M0: byte s stands for 2^(s - 127), 255 for NaN).
// Byte j of a row of codes holds value 2j in its low and value 2j + 1 in its
// high half; byte i of a row of scales is the scale of block i.
//
// Quantisation: with t the largest magnitude of the block, s = max(0, 127 +
// floor(log2 t) - 2) (2 is E2M1's largest exponent), so every value divided by
// the scale lies below 8 in magnitude; it rounds to the nearest of the eight
// magnitudes, ties to the even code, and 6 from there on. A block of zeros has
// s = 0; one with an infinity or a NaN has s = 255 and codes 0 and reads as NaN.
// Dividing by a power of two is exact, so the codes are defined to the bit.
//
// The conversions are the gfx950 instructions (two values each, one issue slot
// at the full VALU rate: measured 5.0 cycles against 5.0 of an add), which were
// checked against the definition for all bf16 values and all scales: a code
// times its scale is exact in bf16, so every consumer multiplies true values.
#pragma once

#include "q3_common.h"

namespace q3 {

constexpr int kMxBlock = 32;  // values of one scale

// The fp32 scale operand of the conversions (only its exponent is used; 255
// makes infinity's exponent, which converts to NaN).
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Eight consecutive values from their codes.
__device__ __forceinline__ bf16x8 mx_bf16x8(uint32_t codes, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The larger magnitude as fp32 bits without the sign: ordered as unsigned
// integers, with the infinities and then the NaNs above every finite value.
__device__ __forceinline__ uint32_t mx_magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// Scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  const uint32_t e = top >> 23;  // 127 + floor(log2), 0 for zero and the subnormals
  return e > 2 ? e - 2 : 0;
}

// Eight consecutive values of one block, held by a lane whose three neighbours
// (lane ^ 1, ^ 2, ^ 3) hold the others: their codes; `byte` gets the block's scale.
__device__ __forceinline__ uint32_t mx_quantize8(const float (&v)[8], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, mx_magnitude(v[e]));
  top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
  byte = mx_scale_byte(top);
  const float s = mx_scale(byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
  return byte == 255 ? 0u : c;
}

// Eight values at p (8 bf16 or fp32, 16-byte aligned).
template <typename T>
__device__ __forceinline__ void mx_load8(const T* p, float (&v)[8]) {
  typedef typename Vec16<T>::type VT;
  constexpr int N = Vec16<T>::N;
#pragma unroll
  for (int c = 0; c < 8 / N; ++c) {
    const VT u = reinterpret_cast<const VT*>(p)[c];
#pragma unroll
    for (int e = 0; e < N; ++e) v[c * N + e] = to_f<T>(u[e]);
  }
}

// n consecutive values (a multiple of 32) to bf16.
int mx_expand(const void* codes, const void* scales, bf16* y, int64_t n, hipStream_t st);

// The rows in use of a 4-bit cache to bf16: y holds K, then V, (B, Hkv, rows, D) each. Rows at or past lens[b] +
// len_add are not read; those up to the next multiple of 64 become zeros (a consumer's tile may reach there), those
// behind are not written. V's NaN blocks in rows from lens[b] on become zeros as well. cst / sst: (b, h) strides of K's, then V's codes / scales in bytes.
int mx_expand_cache(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, bf16* y,
                    int64_t B, int64_t Hkv, int64_t rows, int64_t D, const int64_t* cst, const int64_t* sst,
                    const int* lens, int len_add, hipStream_t st);

}  // namespace q3
