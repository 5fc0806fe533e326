// Expert products over 4-bit weights for few rows per slot (decode).
//
// gate-up: act[pos] = silu(W_g x) * (W_u x);  down: y[pair] = W_2 act[pos].
// Weights are MX4 blocks (mx.h), rows bf16, MX8 or MX4.  What bounds it is the
// weights' bytes: each slot's are read once for up to 32 rows (16 where act comes in two
// parts, below).  Measured, weights in no cache, gate-up / down: 7 tokens x 8 of 64 experts,
// 7168 x 2048, MX8 rows 100 / 51 us (at 6.6 / 6.4 TB/s), MX4 rows 99 / 50; 16 x 8 of 128,
// 2048 x 768, drawn unevenly, bf16 rows 14.2 / 10.3 us (62 / 31 MB at 4.3 / 3.0 TB/s: the
// start and the longest slot's passes of so short a kernel), MX4 rows 13.2 / 7.7 (reading 54
// and 33 MB and nothing else takes 9.7 and 6.6 us).  MX4 rows, measured and not kept: the
// first chunk's weights sent before the rows' addresses are known (down 8.4 -> 7.5, gate-up
// of 16 experts of 4096 x 1024 17.3 -> 18.0, elsewhere within 2%), weights a chunk ahead of
// the products (13.7 / 10.0), 2 or 4 chunks at a time.
//
// A workgroup computes 64 weight rows, four 16-row blocks, for one slot: 32 act
// columns (gate and up) or 64 y columns.  Its waves split the row's K between them,
// so that the reads of a short row are all in flight at once: a wave keeps its chunks'
// weights (one contiguous KiB per 16 rows and 128 columns) and row fragments in
// registers, and the waves' partial sums are added in LDS, in wave order.
//
// The matrix instruction's first operand is the weights, so a lane's four
// results are four neighbouring output columns of one row (lane l: row l % 16,
// columns 4 (l / 16)..).  MX4 rows: e2m1 by e2m1, a lane group's 32 columns on either side
// as they lie, one instruction for 128 columns.  MX8 rows: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies
// e2m1 by e4m3 with both groups' scales; its e4m3 operand holds columns 16 g..
// and 64 + 16 g.. of a chunk in lane group g = l / 16, while scales and the e2m1
// operand go by columns 32 g...  It adds the products of 8 neighbouring columns in
// fixed point, cut 13 bits below the largest one's power of two, and those sums in
// f32 (measured; the cut is some 1e-4 of a result, where rounding rows to e4m3
// costs 2.6e-2; f32 outputs of the plain product take two instructions, which lose
// nothing, rows8_part in mx.h).  bf16 rows: the weights become bf16 in registers
// (exactly: two mantissa bits) and feed v_mfma_f32_16x16x32_bf16 four times, step
// j taking columns 32 g + 8 j.. from either side.
#pragma once

#include "mx.h"

namespace lmoe {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8v_t __attribute__((ext_vector_type(8)));

struct Mx4Args {
  const void* a;            // gate-up: rows [T, K]; down: rows [n_pairs, K] in sorted order
  const uint8_t* a_scale;   // MX8 and MX4 rows: [.., K / 32], else null
  const uint8_t* w;
  long long w_slot_bytes;
  int K, N;                 // row length; output columns (I or H)
  int topk, P, n_pairs;
  const int32_t* offsets;
  const int32_t* sorted_pairs;
  const int32_t* active;
  const int32_t* tile_off;
  const int32_t* meta;
  void* out;                // act rows, or y rows by pair
  uint8_t* out_scale;       // act rows in MX8 or MX4
  bool out_f32;             // y in f32
  bool split;               // bf16 act rows in two parts, [.., 2, I]
  int rows;                 // RowKind of a, and of act
};

// One row's share of a 16 x 128 fragment: this lane's 32 values.
template <int R>
struct RowFrag;
template <>
struct RowFrag<kRowsMx8> {
  i32x8_t v;
  int scale;
};
template <>
struct RowFrag<kRowsMx8Parts> : RowFrag<kRowsMx8> {};
template <>
struct RowFrag<kRowsMx4> {
  i32x4_t v;
  int scale;
};
template <>
struct RowFrag<kRowsBf16> {
  i32x4_t v[4];
};

// The fragment of chunk c of the row at p (sp: its scales).  Values past K read
// as zero: the weights' padding is zero, but zero times a stray NaN is not.
template <int R>
__device__ __forceinline__ RowFrag<R> load_row_frag(const char* p, const uint8_t* sp, int c, int K,
                                                    int g) {
  RowFrag<R> f;
  const int k0 = c * kMxChunk;
  const i32x4_t zero = {0, 0, 0, 0};
  if constexpr (R == kRowsMx4) {
    const bool in = k0 + 32 * g < K;
    f.v = *reinterpret_cast<const i32x4_t*>(p + (in ? (k0 >> 1) + 16 * g : 0));
    const int s = sp[in ? 4 * c + g : 0];
    if (!in) f.v = zero;
    f.scale = in ? s : kScaleOne;
  } else if constexpr (holds_mx8(R)) {
    const bool lo = k0 + 16 * g < K, hi = k0 + 64 + 16 * g < K, sc = k0 + 32 * g < K;
    i32x4_t a = *reinterpret_cast<const i32x4_t*>(p + (lo ? k0 + 16 * g : 0));
    i32x4_t b = *reinterpret_cast<const i32x4_t*>(p + (hi ? k0 + 64 + 16 * g : 0));
    const int s = sp[sc ? 4 * c + g : 0];
    if (!lo) a = zero;
    if (!hi) b = zero;
    f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    f.scale = sc ? s : kScaleOne;
  } else {
    const bool in = k0 + 32 * g < K;
    const char* q = p + (in ? 2 * (k0 + 32 * g) : 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f.v[j] = *reinterpret_cast<const i32x4_t*>(q + 16 * j);
      if (!in) f.v[j] = zero;
    }
  }
  return f;
}

// Eight weights (one dword) as bf16, times 2^e.
__device__ __forceinline__ bf16x8v_t weights_bf16(int word, float s) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 0);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 1);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 2);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 3);
  return bf16x8v_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// acc += W x^T of one chunk: 16 weight rows, 16 rows.  Byte B of scale: the
// weights' scale.
template <int R, int B = 0>
__device__ __forceinline__ f32x4_t mx4_step(i32x4_t w, int scale, const RowFrag<R>& x, f32x4_t acc) {
  if constexpr (R == kRowsMx4) {
    const i32x8_t wide = __builtin_shufflevector(w, w, 0, 1, 2, 3, 0, 1, 2, 3);
    const i32x8_t row = __builtin_shufflevector(x.v, x.v, 0, 1, 2, 3, 0, 1, 2, 3);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide, row, acc, 4 /* e2m1 */, 4, B, scale, 0, x.scale);
  } else if constexpr (R == kRowsMx8) {
    const i32x8_t wide = __builtin_shufflevector(w, w, 0, 1, 2, 3, 0, 1, 2, 3);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide, x.v, acc, 4 /* e2m1 */, 0 /* e4m3 */, B,
                                                            scale, 0, x.scale);
  } else if constexpr (R == kRowsMx8Parts) {
    const i32x8_t wide = __builtin_shufflevector(w, w, 0, 1, 2, 3, 0, 1, 2, 3);
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide, rows8_part<false>(x.v), acc, 4, 0, B, scale, 0, x.scale);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide, rows8_part<true>(x.v), acc, 4, 0, B, scale, 0, x.scale);
  } else {
    const float s = mx_scale_f32((scale >> (8 * B)) & 255);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(weights_bf16(w[j], s), __builtin_bit_cast(bf16x8v_t, x.v[j]),
                                                    acc, 0, 0, 0);
    return acc;
  }
}

// A lane's results are columns 4 g.. and 16 + 4 g.. of 32 (g = lane / 16): two short
// runs.  Lane groups 2 q and 2 q + 1 trade one each, so that a lane holds eight
// neighbouring columns, from joined_column on, and a row leaves in half as many
// pieces (32768 rows of 2048 columns, down product of 768: 146 -> 132 us from bf16
// rows, 119.5 -> 106 from MX8 rows).
__device__ __forceinline__ void join_columns(uint32_t& lo, uint32_t& hi) {
  float a = __uint_as_float(lo), b = __uint_as_float(hi);
  permlane_swap<16>(a, b);
  lo = __float_as_uint(a);
  hi = __float_as_uint(b);
}
__device__ __forceinline__ int joined_column(int lane) { return (lane & 16) + 8 * (lane >> 5); }

// Every lane calls it; p: the row's first of the 32 columns.
__device__ __forceinline__ void store_bf16x8(uint16_t* p, int lane, bool live, const f32x4_t lo, const f32x4_t hi) {
  uint32_t a = pack_bf16x2(lo[0], lo[1]), b = pack_bf16x2(lo[2], lo[3]);
  uint32_t c = pack_bf16x2(hi[0], hi[1]), d = pack_bf16x2(hi[2], hi[3]);
  join_columns(a, c);
  join_columns(b, d);
  if (live) *reinterpret_cast<uint4*>(p + joined_column(lane)) = make_uint4(a, b, c, d);
}

// act = silu(gate) * up of eight columns of one row, held by the four lanes
// l, l ^ 16, l ^ 32, l ^ 48 (lane group g: columns i0 + 4 g.. and i0 + 16 + 4 g..
// of a group of 32): stored in bf16, or in MX8 or MX4 with the group's scale.
template <int R>
__device__ __forceinline__ void store_act(const Mx4Args& g, int pos, int i0, int lane, bool live,
                                          const f32x4_t (&gate)[2], const f32x4_t (&up)[2]) {
  const int col = 4 * (lane >> 4);
  float v[2][4];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[p][e] = silu_f32(gate[p][e]) * up[p][e];
  size_t row = static_cast<size_t>(pos) * g.N;
  if constexpr (R != kRowsBf16) {
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = umax32(m, abs_bits(v[p][e]));
    float a = __uint_as_float(m), b = a;
    permlane_swap<16>(a, b);
    m = umax32(__float_as_uint(a), __float_as_uint(b));
    a = b = __uint_as_float(m);
    permlane_swap<32>(a, b);
    const float amax = __uint_as_float(umax32(__float_as_uint(a), __float_as_uint(b)));
    const int byte = R == kRowsMx8 ? mx8_scale_byte(amax) : mx4_scale_byte(amax);
    const float s = mx_scale_f32(byte);
    uint32_t lo, hi;
    if constexpr (R == kRowsMx8) {
      lo = pack_e4m3x4(v[0][0], v[0][1], v[0][2], v[0][3], s);
      hi = pack_e4m3x4(v[1][0], v[1][1], v[1][2], v[1][3], s);
    } else {
      lo = pack_e2m1x4(v[0][0], v[0][1], v[0][2], v[0][3], s, byte);
      hi = pack_e2m1x4(v[1][0], v[1][1], v[1][2], v[1][3], s, byte);
    }
    join_columns(lo, hi);
    if (live) {
      uint8_t* out = static_cast<uint8_t*>(g.out);
      const size_t at = row + i0 + joined_column(lane);
      if constexpr (R == kRowsMx8) *reinterpret_cast<uint2*>(out + at) = make_uint2(lo, hi);
      else *reinterpret_cast<uint32_t*>(out + at / 2) = lo | hi << 16;
      if (col == 0)
        g.out_scale[static_cast<size_t>(pos) * (g.N / kMxGroup) + i0 / kMxGroup] = static_cast<uint8_t>(byte);
    }
  } else {
    if (g.split) row *= 2;
    uint16_t* out = static_cast<uint16_t*>(g.out) + row + i0;
    store_bf16x8(out, lane, live, f32x4_t{v[0][0], v[0][1], v[0][2], v[0][3]},
                 f32x4_t{v[1][0], v[1][1], v[1][2], v[1][3]});
    if (g.split) {  // what the rounding left, none of what is not finite
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float hi = bf16lo(pack_bf16x2(v[p][e], 0.0f));
          v[p][e] = fabsf(hi) < __builtin_inff() ? v[p][e] - hi : 0.0f;
        }
      store_bf16x8(out + g.N, lane, live, f32x4_t{v[0][0], v[0][1], v[0][2], v[0][3]},
                   f32x4_t{v[1][0], v[1][1], v[1][2], v[1][3]});
    }
  }
}

// This lane's columns of one y row: n + 4 g.. (lo) and n + 16 + 4 g.. (hi).
__device__ __forceinline__ void store_y(const Mx4Args& g, int pair, int n, int lane, bool live, const f32x4_t lo,
                                        const f32x4_t hi) {
  const size_t at = static_cast<size_t>(pair) * g.N + n;
  if (g.out_f32) {
    if (live) {
      float* p = static_cast<float*>(g.out) + at + 4 * (lane >> 4);
      *reinterpret_cast<f32x4_t*>(p) = lo;
      *reinterpret_cast<f32x4_t*>(p + 16) = hi;
    }
  } else {
    store_bf16x8(static_cast<uint16_t*>(g.out) + at, lane, live, lo, hi);
  }
}

// Waves of a workgroup.  Past one token there are workgroups enough, and four waves
// with twice the work each are ahead of eight (us, gate-up / down of bf16 rows, four against
// eight): 16 tokens x 8 over 128 experts of 2048 x 768 15.2 / 10.8 against 16.4 / 12.4,
// 7 x 8 over 64 of 7168 x 2048 96.0 / 47.7 against 95.0 / 50.9, 61 x 4 over 60 of 2048 x 1408
// 34.6 / 20.7 against 36.6 / 23.4, 40 x 4 over 64 of 1024 x 512 8.9 / 6.1 against 10.5 / 7.5;
// eight are ahead where workgroups are few and rows long, 16 x 2 over 16 of 4096 x 1024 17.4 /
// 8.9 against 15.3 / 9.4 (MX8 and MX4 rows 14.3 / 8.1 against 14.0 / 8.9).  One token has few,
// and short ones.
constexpr int kFewMxWaves = 4;
constexpr int kOneMxWaves = 8;
constexpr int kFewMxBlocks = 4;  // 16-row weight blocks of a workgroup
constexpr int kFewMxRows = 32;   // rows of one pass over a slot's weights

// act rows of a few tokens are kept in two bf16 parts, high and low, 16 bits in all:
// where one token's output hangs on a few act values, their rounding to bf16 does not
// average out (one token's error against 64 bits was 1.4 to 1.6 times that of the
// output's own rounding).  Up to eight rows the parts are rows r and r + 8 of one
// fragment, which multiplies sixteen rows anyway; past that they are two fragments,
// sixteen rows a pass.  The parts' sums are added last, so a row's bits are the same.
// Row tiles keep one bf16 part: two would double the down product, which the matrix
// units bound in tall tiles, and short ones, which weights bound, take the same form so
// that a row's bits do not depend on its tile's height.  The price is act's rounding in
// every output: its error is 1.41 times the output's own rounding (1.35 to 1.46 over 160
// layers of 9 to 200 tokens), whatever rows are beside it.
constexpr int kFewMxSplitRows = 16;

// the other half of sixteen lanes: lane l from lane l ^ 8
__device__ __forceinline__ f32x4_t other_part(const f32x4_t v) {
  return f32x4_t{dpp_f32<kDppRowRor8>(v[0]), dpp_f32<kDppRowRor8>(v[1]), dpp_f32<kDppRowRor8>(v[2]),
                 dpp_f32<kDppRowRor8>(v[3])};
}

// Chunks [c0, c1) of RB weight blocks by NF row fragments, U chunks' loads at a time.
// (blocks: how many of the RB there are; the last stands in for the others)
// A quad's scales come as one dword, not as a byte at each chunk, which saves a third of the
// loads.  CARRY: at the quad's first chunk, and kept: 16 tokens x 8 of 128 experts, 2048 x
// 768, gate-up / down of bf16 rows 15.8 / 10.7 -> 14.2 / 10.3 us, MX8 rows 15.4 / 10.6 -> 13.8
// / 9.4, MX4 rows 13.7 / 8.9 -> 13.1 / 7.8.  Else once a round, twice where a round's chunks
// lie in two quads: where a few waves each have little more than one round, the test of a
// quad's start would cut it in two (one token of 2048 x 768 and of 7168 x 2048, bf16 rows
// 12.4 -> 11.6 and 50.5 -> 47.0 us, MX8 rows 10.5 -> 10.2, 41.0 -> 37.9, MX4 rows 10.2 -> 9.8,
// 37.4 -> 35.0; kept, MX8 rows 11.1 and 38.8).
template <int R, int RB, int NF, int U, bool CARRY>
__device__ __forceinline__ void few_chunks(const uint8_t* wblk, int bb, int blocks, int K, int c0, int c1, int lane,
                                           const char* const (&row)[NF], const uint8_t* const (&row_scale)[NF],
                                           f32x4_t (&acc)[RB][NF]) {
  auto scales_of = [&](const uint8_t* quad, int b) {
    return *reinterpret_cast<const int*>(quad + min(b, blocks - 1) * bb + lane * 4);
  };
  int quad_sc[RB], next_sc[RB];
  for (int c = c0; c < c1; c += U) {
    i32x4_t w[U][RB];
    int sc[U][RB];
    RowFrag<R> x[U][NF];
    const int first = c >> 2;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u > 0 && c + u >= c1) break;
      const uint8_t* quad = wblk + ((c + u) >> 2) * kMxQuadBytes;
      const int byte = (c + u) & 3;
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const uint8_t* p = quad + min(b, blocks - 1) * bb;
        w[u][b] = __builtin_nontemporal_load(reinterpret_cast<const i32x4_t*>(p + 256 + byte * 1024 + lane * 16));
      }
      if (CARRY ? c + u == c0 || byte == 0 : u == 0) {
#pragma unroll
        for (int b = 0; b < RB; ++b) quad_sc[b] = scales_of(quad, b);
      }
      if constexpr (CARRY) {
#pragma unroll
        for (int b = 0; b < RB; ++b) sc[u][b] = quad_sc[b];
      }
#pragma unroll
      for (int f = 0; f < NF; ++f) x[u][f] = load_row_frag<R>(row[f], row_scale[f], c + u, K, lane >> 4);
    }
    if constexpr (!CARRY) {
      const int last = (min(c + U, c1) - 1) >> 2;
      if (last != first) {
#pragma unroll
        for (int b = 0; b < RB; ++b) next_sc[b] = scales_of(wblk + last * kMxQuadBytes, b);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u > 0 && c + u >= c1) break;
      const bool next = (c + u) >> 2 != first;
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const int scale = (CARRY ? sc[u][b] : next ? next_sc[b] : quad_sc[b]) >> (8 * ((c + u) & 3));
#pragma unroll
        for (int f = 0; f < NF; ++f) acc[b][f] = mx4_step<R>(w[u][b], scale, x[u][f], acc[b][f]);
      }
    }
  }
}

// NF 16-row fragments of rows [p0, p0 + rows) of one slot.  ONE: the one token's
// act row p0.  SP: rows in two parts, see above.  pairs: the rows' pairs; act rows lie
// from p0 on, or (SCAN) each at its pair.
template <bool GU, int R, int NF, int NW, bool ONE, bool SP, bool SCAN>
__device__ __forceinline__ void few_rows(const Mx4Args& g, const uint8_t* wblk, int blocks, int cb, int p0, int rows,
                                         const int32_t* pairs, f32x4_t* s_part) {
  constexpr int RB = kFewMxBlocks;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunks = mx4_chunks(g.K);
  const char* row[NF];
  const uint8_t* row_scale[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int r = !SP ? 16 * f + (lane & 15) : NF == 1 ? lane & 7 : lane & 15;
    const int at = r < rows ? r : 0;
    size_t src = ONE ? 0 : GU ? pairs[at] / g.topk : SCAN ? pairs[at] : p0 + at;
    if constexpr (SP) src = 2 * src + (NF == 1 ? (lane >> 3) & 1 : f);
    row[f] = static_cast<const char*>(g.a) + row_bytes<R>(src, g.K);
    row_scale[f] = R != kRowsBf16 ? g.a_scale + src * (g.K / kMxGroup) : nullptr;
  }
  f32x4_t acc[RB][NF];
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[b][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  few_chunks<R, RB, NF, ONE ? 2 : 1, !ONE>(wblk, mx4_block_bytes(g.K), blocks, g.K, wave * chunks / NW,
                                           (wave + 1) * chunks / NW, lane, row, row_scale, acc);
  // partial sums of a fragment, [wave][block][lane], added in wave order
  f32x4_t high[2];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    if (f > 0) __syncthreads();  // the last fragment's sums have been read
#pragma unroll
    for (int b = 0; b < RB; ++b) s_part[(wave * RB + b) * 64 + lane] = acc[b][f];
    __syncthreads();
    // gate-up: one wave, which has the 32 columns of a scale; down: a wave for 32 columns
    if (wave >= (GU ? 1 : RB / 2)) continue;
    constexpr int TB = GU ? RB : 2;
    const int b0 = GU ? 0 : 2 * wave;
    f32x4_t t[TB];
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      t[b] = s_part[(b0 + b) * 64 + lane];
#pragma unroll
      for (int v = 1; v < NW; ++v) t[b] += s_part[(v * RB + b0 + b) * 64 + lane];
    }
    if constexpr (SP) {
      if constexpr (NF == 1) {
        t[0] += other_part(t[0]);
        t[1] += other_part(t[1]);
      } else {
        if (f == 0) {
          high[0] = t[0];
          high[1] = t[1];
          continue;
        }
        t[0] = high[0] + t[0];
        t[1] = high[1] + t[1];
      }
    }
    const int r = SP ? lane & 15 : 16 * f + (lane & 15);
    const bool live = r < rows;  // of eight rows at most, those in the lower lanes
    if constexpr (GU) {
      const f32x4_t gate[2] = {t[0], t[2]}, up[2] = {t[1], t[3]};
      store_act<R>(g, SCAN ? (live ? pairs[r] : 0) : p0 + r, cb * 32, lane, live, gate, up);
    } else if (b0 < blocks) {
      store_y(g, live ? pairs[r] : 0, cb * 64 + 32 * wave, lane, live, t[0], t[1]);
    }
  }
}

// The ids of a call that builds no permutation.  A pair whose expert the bank's table
// leaves out may have it in a second bank (the decode overflow buffer, one token only).
struct TokenIds {
  const int32_t* ids;
  const int32_t* log2phy;  // or null: ids are slots
  int n_log2phy;
  const uint8_t* w_b;      // the second bank, or null
  const int32_t* log2phy_b;
  int n_log2phy_b, P_b;
};
__device__ __forceinline__ int slot_of_id(const TokenIds& o, int P, int e) {  // or -1
  int s = e;
  if (o.log2phy != nullptr) s = e >= 0 && e < o.n_log2phy ? o.log2phy[e] : -1;
  return s >= 0 && s < P ? s : -1;
}

// Few tokens straight from their ids: a lane looks a pair's slot up, and a workgroup
// whose pair is the first of its slot takes all of the slot's pairs, in order.  The
// permutation's launch and its three dependent loads (slot, offset, pair) become two
// (id, table): two tokens of the 2048 x 768 layer 26.0 -> 23.0 us.  (A list of up to
// 1024 ids in LDS, scanned by every workgroup, cost what it saved from 32 pairs on.)
// Returns the pairs (0: another workgroup has them), the same for the
// whole workgroup.
constexpr int kScanMaxPairs = 64;
__device__ __forceinline__ int scan_pairs(const Mx4Args& g, const TokenIds& o, int32_t* s_pairs, int* slot) {
  const int lane = threadIdx.x & 63;
  const int mine = lane < g.n_pairs ? slot_of_id(o, g.P, o.ids[lane]) : -1;
  const int s = read_lane_i32(mine, blockIdx.y);
  if (s < 0) return 0;
  const uint64_t m = __ballot(mine == s);
  if (__builtin_ctzll(m) != static_cast<int>(blockIdx.y)) return 0;
  if (mine == s && threadIdx.x < 64) s_pairs[__popcll(m & ((1ull << lane) - 1))] = lane;
  __syncthreads();
  *slot = s;
  return __popcll(m);
}

// (column block, active slot) of a grid of [ceil(N / 32 or 64), slots]; SCAN: (column
// block, pair)
template <bool GU, int R, bool SP, bool SCAN>
__global__ __launch_bounds__(kFewMxWaves * 64) void mx4_few_kernel(Mx4Args g, TokenIds o) {
  __shared__ f32x4_t s_part[kFewMxWaves * kFewMxBlocks * 64];
  __shared__ int32_t s_pairs[SCAN ? kScanMaxPairs : 1];
  int slot, p0, p1;
  if constexpr (SCAN) {
    p0 = 0;
    p1 = scan_pairs(g, o, s_pairs, &slot);
    if (p1 == 0) return;
  } else {
    slot = g.active[blockIdx.y];
    if (slot < 0) return;
    p0 = g.offsets[slot];
    p1 = g.offsets[slot + 1];
  }
  const int32_t* pairs = SCAN ? s_pairs : g.sorted_pairs;
  const int cb = blockIdx.x;
  const int blocks = min(kFewMxBlocks, (GU ? 2 * g.N : g.N) / 16 - cb * kFewMxBlocks);
  const uint8_t* wblk = g.w + slot * g.w_slot_bytes + static_cast<size_t>(cb) * kFewMxBlocks * mx4_block_bytes(g.K);
  constexpr int PASS = SP ? kFewMxSplitRows : kFewMxRows;
  for (int p = p0; p < p1; p += PASS) {
    const int rows = min(PASS, p1 - p);
    if (p > p0) __syncthreads();  // the last pass's sums have been read
    if (rows > PASS / 2)
      few_rows<GU, R, 2, kFewMxWaves, false, SP, SCAN>(g, wblk, blocks, cb, p, rows, pairs + p, s_part);
    else
      few_rows<GU, R, 1, kFewMxWaves, false, SP, SCAN>(g, wblk, blocks, cb, p, rows, pairs + p, s_part);
  }
}

// ---------------------------------------------------------------------------
// One token: no permutation.  Pair j's expert is looked up where it is needed, its
// act row is row j, and the down product ends in the weighted combine: two launches
// where the permutation, the split-K kernel twice and the combine are four.  Measured,
// both in a graph, 8 experts: 2048 x 768 (13.4 + 6.7 MB: latency of the id, table, weight
// chain) 11.6 us from bf16 rows, 10.3 from MX8 rows, 9.8 from MX4 rows; 7168 x 2048 (125 +
// 62 MB) 47.2 / 37.9 / 35.0.  The down product's waves then add
// their parts of K in another order than the split-K kernel's; the same order, parts
// through LDS, cost a quarter at 7168 x 2048 (the step 51.7 -> 65.0 us).
// ---------------------------------------------------------------------------
__device__ __forceinline__ const uint8_t* expert_of_pair(const Mx4Args& g, const TokenIds& o, int j) {  // or null
  const int e = o.ids[j];
  int s = slot_of_id(o, g.P, e);
  if (s >= 0) return g.w + s * g.w_slot_bytes;
  if (o.w_b == nullptr) return nullptr;
  s = e >= 0 && e < o.n_log2phy_b ? o.log2phy_b[e] : -1;
  return s >= 0 && s < o.P_b ? o.w_b + s * g.w_slot_bytes : nullptr;
}
// the same, known to be the same in every lane
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  typedef const __attribute__((address_space(1))) uint8_t* global_t;  // not flat loads
  return (const uint8_t*)(global_t)(static_cast<uint64_t>(hi) << 32 | lo);
}

template <int R>
__global__ __launch_bounds__(kOneMxWaves * 64) void mx4_one_gateup_kernel(Mx4Args g, TokenIds o) {
  __shared__ f32x4_t s_part[kOneMxWaves * kFewMxBlocks * 64];
  const int j = blockIdx.y;
  const uint8_t* expert = uniform(expert_of_pair(g, o, j));
  if (expert == nullptr) return;
  const int cb = blockIdx.x;
  const uint8_t* wblk = expert + static_cast<size_t>(cb) * kFewMxBlocks * mx4_block_bytes(g.K);
  few_rows<true, R, 1, kOneMxWaves, true, false, false>(g, wblk, kFewMxBlocks, cb, j, 1, nullptr, s_part);
}

// 16 columns of out = add + sum_j w_j W2_j act_j.  The waves take (pair, part of K)
// units in turn, each adding its units' weighted sums; the waves' sums are added in
// order.  A unit is the whole K of a pair where there are eight pairs or more.  bf16
// rows come in two parts, the fragment's lower and upper rows.
template <int R>
__global__ __launch_bounds__(kOneMxWaves * 64) void mx4_one_down_kernel(Mx4Args g, TokenIds o,
                                                                       const uint16_t* __restrict__ wts,
                                                                       const uint16_t* __restrict__ add) {
  constexpr int NW = kOneMxWaves;
  __shared__ f32x4_t s_part[NW * 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int k = g.n_pairs;
  const int chunks = mx4_chunks(g.K);
  const int bb = mx4_block_bytes(g.K);
  const int parts = min((NW + k - 1) / k, chunks);
  f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int u = wave; u < k * parts; u += NW) {
    const int j = u / parts, part = u - j * parts;
    const uint8_t* expert = uniform(expert_of_pair(g, o, j));
    if (expert == nullptr) {  // counted once
      if (blockIdx.x == 0 && part == 0 && lane == 0) add_device_flag(LMOE_FLAG_UNPLACED, 1);
      continue;
    }
    const float wj = bf16_to_f32(wts[j]);
    const size_t src = R != kRowsBf16 ? j : 2 * j + ((lane >> 3) & 1);
    const char* row[1] = {static_cast<const char*>(g.a) + row_bytes<R>(src, g.K)};
    const uint8_t* row_scale[1] = {R != kRowsBf16 ? g.a_scale + static_cast<size_t>(j) * (g.K / kMxGroup) : nullptr};
    f32x4_t acc[1][1] = {{f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}}};
    const uint8_t* wblk = expert + static_cast<size_t>(blockIdx.x) * bb;
    few_chunks<R, 1, 1, 4, false>(wblk, bb, 1, g.K, part * chunks / parts, (part + 1) * chunks / parts, lane, row,
                                  row_scale, acc);
    sum += wj * acc[0][0];
  }
  if constexpr (R == kRowsBf16) sum += other_part(sum);
  // the sixteen rows of the fragment are the same row: lanes 0, 16, 32 and 48 have it
  if ((lane & 15) == 0) s_part[wave * 4 + (lane >> 4)] = sum;
  __syncthreads();
  if (threadIdx.x < 4) {
    const int h = blockIdx.x * 16 + threadIdx.x * 4;
    f32x4_t t = s_part[threadIdx.x];
    for (int v = 1; v < NW; ++v) t += s_part[v * 4 + threadIdx.x];
    if (add != nullptr) {
      const uint2 a = *reinterpret_cast<const uint2*>(add + h);
      t += f32x4_t{bf16lo(a.x), bf16hi(a.x), bf16lo(a.y), bf16hi(a.y)};
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(g.out) + h) =
        make_uint2(pack_bf16x2(t[0], t[1]), pack_bf16x2(t[2], t[3]));
  }
}

}  // namespace lmoe
