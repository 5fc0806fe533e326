// One matrix of 4-bit weights: y = x W^T (+ bias) (+ add).
//
// Rows are bf16, MX8 or MX4; weights one slot of a bank in order (mx.h).  Sums, bias and add
// are in f32 and are rounded once, to out's type; of MX8 rows with a bf16 out the products of
// eight neighbouring columns are added in fixed point first (rows8_part in mx.h).
#pragma once

#include "mx4_few.h"

namespace lmoe {

struct LinearArgs {
  const void* a;            // rows [T, K]
  const uint8_t* a_scale;   // MX8 and MX4 rows, else null
  const uint8_t* w;
  int T, K, N;
  const void* bias;         // [N] bf16 or f32, or null
  const uint16_t* add;      // [T, N] bf16, or null
  void* out;                // [T, N] bf16 or f32
  bool bias_f32, out_f32;
  int xcd_rows;             // row tiles: how many parts the XCDs divide them into
};

// bias and add of four neighbouring columns of a row, in that order.
__device__ __forceinline__ f32x4_t linear_terms(const LinearArgs& g, int row, int n, f32x4_t v) {
  if (g.bias != nullptr) {
    if (g.bias_f32) {
      v += *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(g.bias) + n);
    } else {
      const uint2 b = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g.bias) + n);
      v += f32x4_t{bf16lo(b.x), bf16hi(b.x), bf16lo(b.y), bf16hi(b.y)};
    }
  }
  if (g.add != nullptr) {
    const uint2 a = *reinterpret_cast<const uint2*>(g.add + static_cast<size_t>(row) * g.N + n);
    v += f32x4_t{bf16lo(a.x), bf16hi(a.x), bf16lo(a.y), bf16hi(a.y)};
  }
  return v;
}

// Four neighbouring columns of a row, rounded once.
__device__ __forceinline__ void store_linear4(const LinearArgs& g, int row, int n, f32x4_t v) {
  v = linear_terms(g, row, n, v);
  const size_t at = static_cast<size_t>(row) * g.N + n;
  if (g.out_f32) *reinterpret_cast<f32x4_t*>(static_cast<float*>(g.out) + at) = v;
  else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(g.out) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// This lane's columns of 32 from n on: n + 4 g.. (lo) and n + 16 + 4 g.. (hi; it may be
// past the matrix).  Every lane calls it.
__device__ __forceinline__ void store_linear(const LinearArgs& g, int row, int n, int lane, bool live, f32x4_t lo, f32x4_t hi) {
  const int col = n + 4 * (lane >> 4);
  if (n + 32 > g.N) {  // the last block alone
    if (live) store_linear4(g, row, col, lo);
    return;
  }
  if (live) {
    lo = linear_terms(g, row, col, lo);
    hi = linear_terms(g, row, col + 16, hi);
  }
  const size_t at = static_cast<size_t>(row) * g.N + n;
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

// Few rows: a workgroup takes RB blocks of 16 columns by NF fragments of 16 rows; its NW
// waves split K, U chunks' loads at a time, and their partial sums are added in LDS in wave
// order.  Bound by the weights' bytes and, below some 20 MB of them, by the launch: 1 x 2048 x
// 5120 of MX4 rows 3.9 us (an empty launch 2.1), 1 x 2048 x 50000 11.0 (54 MB; reading them
// and nothing else 9.7), 16 rows there 12.0 (MX4) and 14.3 (bf16).
template <int R, int RB, int NF, int NW, int U>
__global__ __launch_bounds__(NW * 64) void mx4_linear_few_kernel(LinearArgs g) {
  __shared__ f32x4_t s_part[NW * RB * NF * 64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunks = mx4_chunks(g.K);
  const int bb = mx4_block_bytes(g.K);
  const int cols = ((g.N >> 4) + RB - 1) / RB;
  const int group = blockIdx.x / cols, cb = blockIdx.x - group * cols;
  const int t0 = group * (16 * NF);
  const int blocks = min(RB, (g.N >> 4) - cb * RB);
  const uint8_t* wblk = g.w + static_cast<size_t>(cb) * RB * bb;
  const char* row[NF];
  const uint8_t* row_scale[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int r = t0 + 16 * f + (lane & 15);
    const size_t src = r < g.T ? r : t0;
    row[f] = static_cast<const char*>(g.a) + row_bytes<R>(src, g.K);
    row_scale[f] = R != kRowsBf16 ? g.a_scale + src * (g.K / kMxGroup) : nullptr;
  }
  f32x4_t acc[RB][NF];
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[b][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  few_chunks<R, RB, NF, U, R != kRowsMx4 || U == 1>(wblk, bb, blocks, g.K, wave * chunks / NW, (wave + 1) * chunks / NW,
                                                    lane, row, row_scale, acc);
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int f = 0; f < NF; ++f) s_part[((wave * RB + b) * NF + f) * 64 + lane] = acc[b][f];
  __syncthreads();
  for (int u = wave; u < RB * NF; u += NW) {
    const int b = u / NF, f = u - b * NF;
    f32x4_t v = s_part[u * 64 + lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += s_part[(w * RB * NF + u) * 64 + lane];
    const int r = t0 + 16 * f + (lane & 15);
    if (b < blocks && r < g.T) store_linear4(g, r, (cb * RB + b) * 16 + 4 * (lane >> 4), v);
  }
}

}  // namespace lmoe
