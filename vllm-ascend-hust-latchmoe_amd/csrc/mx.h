// Microscaling formats (OCP MX) as this library stores them.
//
// A group of 32 values along a row shares one scale 2^e, held as the byte
// e + 127 (255: every value of the group is NaN).  e is the smallest integer
// that keeps the group's largest magnitude within the element format (448 for
// e4m3, 6 for e2m1), so no value saturates; a group of zeros, or one whose e
// would be lower, has e = -127.  A group that holds a NaN or an infinity, which
// neither element format can scale, is NaN as a whole.
//
// MX8 rows: q [R, K] e4m3 bytes, scale [R, K / 32] bytes, both row-major.
//
// MX4 rows: q [R, K / 2] bytes, two e2m1 values each (the even column in the low half),
// scale [R, K / 32] bytes, both row-major.  A row's 16 bytes of a group are the matrix
// instruction's operand as they lie.
//
// MX4 weights of an [N, K] matrix, in the order the matrix instructions read
// them: N / 16 blocks of 16 rows; a block is a run of quads (512 columns), each
// 256 bytes of scales and then up to four chunks (128 columns) of 1 KiB.  Lane l
// of a wave stands for row l % 16 and the 32 columns from 32 (l / 16) of a
// chunk: its 16 bytes of a chunk are at 16 l (two values per byte, the even
// column in the low half), its scale byte of chunk c of the quad at 4 l + c.
// So a wave's fragment of 16 rows x 128 columns is one contiguous KiB, and a
// block is read front to back.  Columns past K of the last chunk hold zeros
// with scale 1.
#pragma once

#include "lmoe_device.h"

namespace lmoe {

constexpr int kMxGroup = 32;
constexpr int kMxChunk = 128;                 // columns of one fragment
constexpr int kMxQuadBytes = 256 + 4 * 1024;  // scales and four chunks
constexpr int kScaleOne = 127;
// Of the plain product, weights' quantisation and MX4 rows' tiles: a tile's blocks and rows
// (256 x 2^23 values) are then within 32 bits of its first.
constexpr int kMxMaxColumns = 1 << 23;

__host__ __device__ inline int mx4_chunks(int K) { return (K + kMxChunk - 1) / kMxChunk; }
__host__ __device__ inline int mx4_block_bytes(int K) {
  return mx4_chunks(K) * 1024 + (K + 511) / 512 * 256;
}

// Scale byte of a group whose largest magnitude is amax, for an element format
// whose largest value is top = (1 + top_frac / 2^23) * 2^top_exp: with amax =
// (1 + f) 2^x the smallest e is x - top_exp, plus one where f > top_frac.  A
// subnormal amax (x < -126) ends at e = -127 either way.
template <int TOP_EXP, uint32_t TOP_FRAC>
__device__ __forceinline__ int mx_scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);  // amax >= 0 or NaN
  const int x = static_cast<int>(u >> 23);   // biased by 127
  const int e = x - TOP_EXP + ((u & 0x7fffffu) > TOP_FRAC ? 1 : 0);
  return x == 255 ? 255 : (e > 0 ? e : 0);
}
__device__ __forceinline__ int mx8_scale_byte(float amax) {
  return mx_scale_byte<8, 0x600000u>(amax);  // 448 = 1.75 * 2^8
}

// 2^e of a scale byte as f32 bits e + 127 in the exponent.  Byte 0 (2^-127) is
// 0.0 here and byte 255 an infinity: the scaled conversions read only the
// exponent field, and take 0 as 2^-127 and 255 as NaN (measured).
__device__ __forceinline__ float mx_scale_f32(int byte) {
  return __uint_as_float(static_cast<uint32_t>(byte) << 23);
}

// |v| where NaN and infinities count as more than any number, for a maximum
// that must not lose them (fmaxf drops NaN): compared as unsigned bits.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ int mx4_scale_byte(float amax) {
  return mx_scale_byte<2, 0x400000u>(amax);  // 6 = 1.5 * 2^2
}

// What a product's rows are held in.  kRowsMx8Parts: MX8 rows whose sums are f32's (rows8_part).
enum RowKind : int { kRowsBf16 = 0, kRowsMx8 = 1, kRowsMx4 = 2, kRowsMx8Parts = 3 };
constexpr bool holds_mx8(int rows) { return rows == kRowsMx8 || rows == kRowsMx8Parts; }
// Bytes before row r of K columns.
template <int R>
__host__ __device__ __forceinline__ size_t row_bytes(size_t r, int K) {
  return R == kRowsMx4 ? r * (static_cast<size_t>(K) >> 1) : r * K * (holds_mx8(R) ? 1 : 2);
}

typedef int i32x8_t __attribute__((ext_vector_type(8)));

// One of two parts whose sum is a fragment of e4m3 bytes: the values below 2 (HIGH false)
// or the others, zeros in the place of what the other part has.  The scaled matrix
// instruction adds the products of eight columns in fixed point, cut 13 bits below the
// largest one's power of two, which is that of its factors' exponents (measured).  e2m1 by
// the lower part are multiples of 2^-10 (2^-9 by .5) whose exponents end at 2^2, by the
// upper part multiples of 2^-3 (2^-2 by .5) that end at 2^10: neither loses anything, and two
// instructions give f32's sums (2000 fragments of each of five distributions: off by 0.97 *
// 2^-24 of the magnitudes at most, one instruction by 1400).  Bit 6 is the exponent's
// highest, that of 2.
template <bool HIGH>
__device__ __forceinline__ i32x8_t rows8_part(const i32x8_t v) {
  i32x8_t p;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bit = (static_cast<uint32_t>(v[i]) >> 6) & 0x01010101u;
    const uint32_t high = (bit << 8) - bit;  // the bytes that have it
    p[i] = static_cast<int>(v[i] & (HIGH ? high : ~high));
  }
  return p;
}

typedef short i16x2_t __attribute__((ext_vector_type(2)));

// Four values / 2^e as e4m3 bytes, lowest first, round to nearest even.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d, float scale) {
  i16x2_t r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, r);
}

// Values / 2^e as e2m1 codes, the first in the lowest bits, round to nearest even.  byte:
// the scale's; the codes of a group that is NaN are zeros.
__device__ __forceinline__ uint32_t pack_e2m1x4(float a, float b, float c, float d, float scale, int byte) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, a, b, scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, c, d, scale, 1);
  return byte == 255 ? 0 : r;
}
__device__ __forceinline__ uint32_t pack_e2m1x8(const float (&v)[8], float scale, int byte) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
  return byte == 255 ? 0 : r;
}

}  // namespace lmoe
