// Expert products over 4-bit weights for few rows per slot (decode).
//
// gate-up: act[pos] = silu(W_g x) * (W_u x);  down: y[pair] = W_2 act[pos].
// Weights are MX4 blocks (mx.h), rows bf16 or MX8.  What bounds it is the
// weights' bytes: each slot's are read once for up to 32 rows.
//
// A workgroup computes 32 output columns (gate-up: 32 gate and 32 up weight
// rows, four 16-row blocks; down: two) for one slot.  Its eight waves split the
// row's K between them, so that the reads of a short row are all in flight at
// once: a wave keeps its chunks' weights (one contiguous KiB per 16 rows and
// 128 columns) and row fragments in registers, and the waves' partial sums are
// added in LDS, in wave order.
//
// The matrix instruction's first operand is the weights, so a lane's four
// results are four neighbouring output columns of one row (lane l: row l % 16,
// columns 4 (l / 16)..).  MX8 rows: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies
// e2m1 by e4m3 with both groups' scales; its e4m3 operand holds columns 16 g..
// and 64 + 16 g.. of a chunk in lane group g = l / 16, while scales and the e2m1
// operand go by columns 32 g...  It adds the products of 8 neighbouring columns in
// fixed point, cut 13 bits below the largest one's power of two, and those sums in
// f32 (measured; the cut is some 1e-4 of a result, where rounding rows to e4m3
// costs 2.6e-2).  bf16 rows: the weights become bf16 in registers
// (exactly: two mantissa bits) and feed v_mfma_f32_16x16x32_bf16 four times, step
// j taking columns 32 g + 8 j.. from either side.
#pragma once

#include "mx.h"

namespace lmoe {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8v_t __attribute__((ext_vector_type(8)));

struct Mx4Args {
  const void* a;            // gate-up: rows [T, K]; down: rows [n_pairs, K] in sorted order
  const uint8_t* a_scale;   // MX8 rows: [.., K / 32], else null
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
  uint8_t* out_scale;       // act rows in MX8
  bool out_f32;             // y in f32
};

// One row's share of a 16 x 128 fragment: this lane's 32 values.
template <bool A8>
struct RowFrag;
template <>
struct RowFrag<true> {
  i32x8_t v;
  int scale;
};
template <>
struct RowFrag<false> {
  i32x4_t v[4];
};

// The fragment of chunk c of the row at p (sp: its scales).  Values past K read
// as zero: the weights' padding is zero, but zero times a stray NaN is not.
template <bool A8>
__device__ __forceinline__ RowFrag<A8> load_row_frag(const char* p, const uint8_t* sp, int c, int K,
                                                     int g) {
  RowFrag<A8> f;
  const int k0 = c * kMxChunk;
  const i32x4_t zero = {0, 0, 0, 0};
  if constexpr (A8) {
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
template <bool A8, int B = 0>
__device__ __forceinline__ f32x4_t mx4_step(i32x4_t w, int scale, const RowFrag<A8>& x, f32x4_t acc) {
  if constexpr (A8) {
    const i32x8_t wide = __builtin_shufflevector(w, w, 0, 1, 2, 3, 0, 1, 2, 3);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide, x.v, acc, 4 /* e2m1 */, 0 /* e4m3 */, B,
                                                            scale, 0, x.scale);
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
// pieces (4096 x 8 rows of 2048 columns: down product 138 -> 113 us).
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
// of a group of 32): stored in bf16, or in MX8 with the group's scale.
template <bool A8>
__device__ __forceinline__ void store_act(const Mx4Args& g, int pos, int i0, int lane, bool live,
                                          const f32x4_t (&gate)[2], const f32x4_t (&up)[2]) {
  const int col = 4 * (lane >> 4);
  float v[2][4];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[p][e] = silu_f32(gate[p][e]) * up[p][e];
  const size_t row = static_cast<size_t>(pos) * g.N;
  if constexpr (A8) {
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
    const int byte = mx8_scale_byte(__uint_as_float(umax32(__float_as_uint(a), __float_as_uint(b))));
    const float s = mx_scale_f32(byte);
    uint32_t lo = pack_e4m3x4(v[0][0], v[0][1], v[0][2], v[0][3], s);
    uint32_t hi = pack_e4m3x4(v[1][0], v[1][1], v[1][2], v[1][3], s);
    join_columns(lo, hi);
    if (live) {
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(g.out) + row + i0 + joined_column(lane)) = make_uint2(lo, hi);
      if (col == 0)
        g.out_scale[static_cast<size_t>(pos) * (g.N / kMxGroup) + i0 / kMxGroup] = static_cast<uint8_t>(byte);
    }
  } else {
    store_bf16x8(static_cast<uint16_t*>(g.out) + row + i0, lane, live, f32x4_t{v[0][0], v[0][1], v[0][2], v[0][3]},
                 f32x4_t{v[1][0], v[1][1], v[1][2], v[1][3]});
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

constexpr int kFewMxWaves = 8;
constexpr int kFewMxRows = 32;  // rows of one pass over a slot's weights

// NF 16-row fragments of rows [p0, p0 + rows) of one slot.
template <bool GU, bool A8, int NF>
__device__ __forceinline__ void few_rows(const Mx4Args& g, const uint8_t* wblk, int cb, int p0, int rows,
                                         f32x4_t* s_part) {
  constexpr int RB = GU ? 4 : 2;
  constexpr int NW = kFewMxWaves;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lg = lane >> 4;
  const int chunks = mx4_chunks(g.K);
  const int bb = mx4_block_bytes(g.K);
  const char* row[NF];
  const uint8_t* row_scale[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int r = 16 * f + (lane & 15);
    const int pos = p0 + (r < rows ? r : 0);
    const size_t src = GU ? g.sorted_pairs[pos] / g.topk : pos;
    row[f] = static_cast<const char*>(g.a) + src * g.K * (A8 ? 1 : 2);
    row_scale[f] = A8 ? g.a_scale + src * (g.K / kMxGroup) : nullptr;
  }
  f32x4_t acc[RB][NF];
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[b][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int c1 = (wave + 1) * chunks / NW;
#pragma unroll 2
  for (int c = wave * chunks / NW; c < c1; ++c) {
    i32x4_t w[RB];
    int sc[RB];
    const uint8_t* quad = wblk + (c >> 2) * kMxQuadBytes;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const uint8_t* p = quad + b * bb;
      w[b] = __builtin_nontemporal_load(
          reinterpret_cast<const i32x4_t*>(p + 256 + (c & 3) * 1024 + lane * 16));
      sc[b] = p[lane * 4 + (c & 3)];
    }
    RowFrag<A8> x[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) x[f] = load_row_frag<A8>(row[f], row_scale[f], c, g.K, lg);
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int f = 0; f < NF; ++f) acc[b][f] = mx4_step<A8>(w[b], sc[b], x[f], acc[b][f]);
  }
  // partial sums, [wave][block][fragment][lane], added in wave order
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int f = 0; f < NF; ++f) s_part[((wave * RB + b) * NF + f) * 64 + lane] = acc[b][f];
  __syncthreads();
  if (wave < NF) {
    const int f = wave;
    f32x4_t t[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      t[b] = s_part[(b * NF + f) * 64 + lane];
      for (int v = 1; v < NW; ++v) t[b] += s_part[((v * RB + b) * NF + f) * 64 + lane];
    }
    const int r = 16 * f + (lane & 15);
    const bool live = r < rows;
    if constexpr (GU) {
      const f32x4_t gate[2] = {t[0], t[2]}, up[2] = {t[1], t[3]};
      store_act<A8>(g, p0 + r, cb * 32, lane, live, gate, up);
    } else {
      store_y(g, live ? g.sorted_pairs[p0 + r] : 0, cb * 32, lane, live, t[0], t[1]);
    }
  }
}

template <bool GU, bool A8>
__global__ __launch_bounds__(kFewMxWaves * 64) void mx4_few_kernel(Mx4Args g) {
  constexpr int RB = GU ? 4 : 2;
  __shared__ f32x4_t s_part[kFewMxWaves * RB * (kFewMxRows / 16) * 64];
  const int slot = g.active[blockIdx.y];
  if (slot < 0) return;
  const int p0 = g.offsets[slot], p1 = g.offsets[slot + 1];
  const int cb = blockIdx.x;
  const uint8_t* wblk = g.w + slot * g.w_slot_bytes + static_cast<size_t>(cb) * RB * mx4_block_bytes(g.K);
  for (int p = p0; p < p1; p += kFewMxRows) {
    const int rows = min(kFewMxRows, p1 - p);
    if (p > p0) __syncthreads();  // the last pass's sums have been read
    if (rows > 16) few_rows<GU, A8, 2>(g, wblk, cb, p, rows, s_part);
    else few_rows<GU, A8, 1>(g, wblk, cb, p, rows, s_part);
  }
}

}  // namespace lmoe
