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

typedef short i16x2_t __attribute__((ext_vector_type(2)));

// Four values / 2^e as e4m3 bytes, lowest first, round to nearest even.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d, float scale) {
  i16x2_t r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, r);
}

}  // namespace lmoe
