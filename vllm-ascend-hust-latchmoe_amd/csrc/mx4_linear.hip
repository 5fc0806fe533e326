// Entry point of the product with one matrix of 4-bit weights.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gemm_lds.h"
#include "mx_tile.h"
#include "mx4_tile.h"
#include "spans.h"

namespace lmoe {

template <int R, int RB, int NF, int NW, int U>
static int launch_few(const LinearArgs& g, hipStream_t stream) {
  const long long grid = (g.N / 16 + RB - 1) / RB * ((g.T + 16ll * NF - 1) / (16 * NF));
  if (grid > 0x7fffffffll) return LMOE_ERR_SHAPE;
  mx4_linear_few_kernel<R, RB, NF, NW, U><<<static_cast<unsigned>(grid), NW * 64, 0, stream>>>(g);
  LMOE_RETURN_LAUNCH();
}

// Workgroups of tiles of BM rows by BN columns.
static long long tiles_of(const LinearArgs& g, long long BM, long long BN) {
  return (g.T + BM - 1) / BM * ((g.N + BN - 1) / BN);
}

// A workgroup's rows and columns.  split_k: its waves split K (mx4_linear_few_kernel), else
// a row tile.
struct LinearForm {
  int rows, cols;
  bool split_k;
};

// Row tiles: the shape with the least time by this measure, in tenths of a us: for each
// round of the workgroups that a CU has at once `round`, and for each of its chunks of K the
// time of 1, 2, .. of them (the last round may have fewer).  A CU's workgroups are those of
// the XCD that has most: 2839 x 6752 x 5136 in tiles of 256 x 256 are 252, but 33 of one XCD's
// 32 CUs, and take 1.7 times what tiles of 128 x 256 do.  The constants are fitted to 900
// random products of 100 to 5000 rows, 512 to 7360 columns and 640 to 9600 outputs, whose
// chosen form takes 1.003 to 1.007 of the best one's time on average (before the XCDs were
// counted: 1.015 to 1.04).  The figures below are
// us of 20 calls in a row, of random values, the shapes in turn (a card that comes from
// lighter work runs the largest up to 10% faster).
struct ShapeCost {
  int BM, BN, at_once, round;
  double chunk[4];
};
// MX4 rows, 256 x 256 / 128 x 128 / 64 x 128 / 64 x 64 tiles:
//   4096 x 7168 x 7168  112 / 143 / 181 / 256      512 x 7168 x 7168   44.3 / 23.8 / 25.1 / 32.0
//   4096 x 2048 x 5120  40.0 / 35.4 / 40.6 / 48.7  300 x 2048 x 5120   18.4 / 10.1 / 8.2 / 8.1
//   2048 x 7168 x 7168  56.7 / 73.8 / 83.5 / 114   300 x 1408 x 2048   15.1 / 8.7 / 6.8 / 5.6
//   1024 x 7168 x 7168  48.5 / 37.5 / 47.0 / 55.2  1000 x 2048 x 2048  18.2 / 10.5 / 8.5 / 8.5
constexpr ShapeCost kShapes4[4] = {{256, 256, 1, 74, {7.8}}, {128, 128, 2, 49, {3.5, 6.1}},
                                   {64, 128, 3, 37, {3.0, 3.9, 5.7}}, {64, 64, 4, 29, {2.5, 3.4, 4.2, 5.5}}};
// MX8 rows, 256 x 256 / 128 x 256 / 128 x 128 / 64 x 128 / 64 x 64 tiles:
//   4096 x 7168 x 7168  167 / 186 / 199 / 246 / 437       512 x 7168 x 7168   73.1 / 40.8 / 36.7 / 31.0 / 41.4
//   4096 x 2048 x 5120  59.4 / 53.4 / 48.1 / 58.3 / 70.1  300 x 2048 x 5120   26.0 / 15.6 / 12.9 / 9.1 / 9.5
//   2048 x 7168 x 7168  90.7 / 94.4 / 104 / 109 / 149     300 x 1408 x 2048   21.0 / 12.2 / 10.4 / 7.3 / 6.1
//   1024 x 7168 x 7168  81.1 / 47.0 / 52.8 / 62.2 / 73.4  1000 x 2048 x 2048  25.8 / 15.7 / 13.3 / 9.4 / 9.8
constexpr ShapeCost kShapes8[5] = {{256, 256, 1, 87, {13.4}}, {128, 256, 1, 53, {6.8}}, {128, 128, 2, 40, {6.4, 9.7}},
                                   {64, 128, 2, 42, {3.2, 4.4}}, {64, 64, 3, 35, {2.5, 3.8, 5.1}}};
// MX8 rows with f32 outputs, in two parts (twice the products; tiles of 256 x 256 spill 112
// registers, those of 128 x 256 are no faster anywhere), 128 x 128 / 64 x 128 / 64 x 64 tiles:
//   4096 x 7168 x 7168  341 / 375 / 487     512 x 7168 x 7168   63.4 / 51.2 / 67.0
//   4096 x 2048 x 5120  81.1 / 87.5 / 106   300 x 2048 x 5120   21.9 / 14.1 / 14.2
//   2048 x 7168 x 7168  188 / 182 / 236     300 x 1408 x 2048   16.8 / 10.6 / 8.5
//   1024 x 7168 x 7168  91.7 / 96.1 / 111   1000 x 2048 x 2048  22.1 / 14.6 / 15.0
constexpr ShapeCost kShapes8Parts[3] = {{128, 128, 2, 66, {9.7, 15.5}}, {64, 128, 2, 40, {5.5, 8.0}},
                                        {64, 64, 3, 38, {4.4, 5.5, 7.3}}};
// bf16 rows, 128 x 256 / 64 x 256 / 32 x 256 tiles:
//   8192 x 7168 x 7168  607 / 642             1024 x 7168 x 7168  111 / 90.1 / 111
//   4096 x 7168 x 7168  350 / 332 / 396       512 x 7168 x 7168   107 / 73.9 / 57.2
//   4096 x 2048 x 5120  88.8 / 73.6 / 89.4    300 x 2048 x 5120   31.0 / 21.2 / 14.5
//   2048 x 7168 x 7168  169 / 185             4096 x 4096 x 4096  105 / 119
constexpr ShapeCost kShapes16[3] = {{128, kTileCols, 2, 32, {19.2, 30.7}}, {64, kTileCols, 2, 0, {12.7, 16.5}},
                                    {32, kTileCols, 2, 16, {8.3, 10.0}}};

template <int S>
static LinearForm cheapest(const ShapeCost (&shapes)[S], const LinearArgs& g, int cus) {
  const int chunks = mx4_chunks(g.K), per_xcd = cus < 8 ? 1 : cus / 8;
  int best = 0;
  double least = 0;
  for (int s = 0; s < S; ++s) {
    const ShapeCost& c = shapes[s];
    LinearArgs shared = g;
    const long long each = (linear_grid(&shared, c.BM, c.BN) / 8 + per_xcd - 1) / per_xcd;  // a CU's tiles
    const long long full = each / c.at_once, last = each % c.at_once;
    double time = full * (c.round + chunks * c.chunk[c.at_once - 1]);
    if (last > 0) time += c.round + chunks * c.chunk[last - 1];
    if (s == 0 || time < least) {
      best = s;
      least = time;
    }
  }
  return {shapes[best].BM, shapes[best].BN, false};
}

// Split K while that makes workgroups enough: for the fewest rows 32 columns by 16 rows a
// workgroup, then 64 by 16, then 64 by 32.  us of these three and of row tiles (T x K x N):
//                 16 x 2048 x 5120   32 x 7168 x 7168     64 x 7168 x 7168     128 x 2048 x 5120
//   MX4 rows      4.4 5.3 5.6  7.0   14.9 11.5 15.2 16.7  25.9 20.3 14.7 17.3   9.4  9.2  9.0  7.5
//   MX8 rows      5.0 5.6 6.1  7.3   17.5 12.5 17.5 17.8  30.4 22.0 17.0 18.2  12.4 10.2 12.0  7.9
//   .. into f32   5.2 5.9 6.8  8.1   17.3 12.5 18.3 26.2  30.2 22.3 18.0 26.7  12.0 10.7 13.3 10.7
//   bf16 rows     5.5 6.5 7.3 13.4   20.1 14.2 20.9 43.6  35.2 24.9 20.8 43.5  16.2 12.2 14.8 13.9
// (bf16 rows' tiles need more workgroups than the others' to be worth it.)
// Past 16384 columns, up to 16 rows, whose rows every workgroup reads again: 128 columns a
// workgroup, a chunk at a time.  us of 32 / 64 / 128 columns:
//                1 x 2048 x 50000    16 x 2048 x 50000   16 x 2048 x 20000  16 x 7168 x 32000
//   MX4 rows     10.9 / 12.4 / 11.0  13.8 / 13.7 / 12.0  7.7 / 8.3 / 7.9    28.5 / 24.1 / 21.5
//   MX8 rows     12.4 / 12.3 / 11.2  15.6 / 14.5 / 12.3  8.5 / 8.6 / 7.7    31.0 / 24.6 / 21.7
//   bf16 rows    15.2 / 13.7 / 12.1  20.5 / 16.8 / 14.3  10.4 / 10.0 / 8.4  36.5 / 27.8 / 23.8
// and below, 8 x 7168 x 16384: 13.2 / 12.9 / 16.4, 14.0 / 13.0 / 16.5, 16.0 / 14.3 / 17.5.
static LinearForm linear_form(int rows, const LinearArgs& g, int cus) {
  if (g.T <= 16 && g.N > 16384) return {16, 128, true};
  if (g.T <= 16 || tiles_of(g, 16, 32) <= cus) return {16, 32, true};
  if (tiles_of(g, 16, 64) <= cus + cus / 4) return {16, 64, true};
  if (tiles_of(g, 32, 64) <= cus) return {32, 64, true};
  if (rows == kRowsMx4) return cheapest(kShapes4, g, cus);
  if (rows == kRowsMx8) return cheapest(kShapes8, g, cus);
  if (rows == kRowsMx8Parts) return cheapest(kShapes8Parts, g, cus);
  if (tiles_of(g, 16, 64) <= 5 * cus / 2) return {16, 64, true};
  return cheapest(kShapes16, g, cus);
}

template <int BM, int CS>
static int launch_rows16(LinearArgs g, long long grid, hipStream_t stream) {
  const int st = launch_tile<Op::kLinear, false, BM, CS>(g, grid, stream);
  if (st != LMOE_OK) return st;
  LMOE_RETURN_LAUNCH();
}

template <int R>
static int launch_linear(LinearArgs g, hipStream_t stream) {
  const int cus = device_cus();
  const LinearForm f = linear_form(R, g, cus);
  auto is = [&](int rows, int cols) { return f.rows == rows && f.cols == cols; };
  if (f.split_k) {
    if (is(16, 128)) return launch_few<R, 8, 1, 8, 1>(g, stream);
    if (is(16, 32)) return launch_few<R, 2, 1, 8, 2>(g, stream);
    if (is(16, 64)) return launch_few<R, 4, 1, 8, 2>(g, stream);
    return launch_few<R, 4, 2, 8, 2>(g, stream);
  }
  if constexpr (R == kRowsMx4) {
    if (is(256, 256)) return launch_mx_linear<Tile4_256x256>(g, stream);
    if (is(128, 128)) return launch_mx_linear<Tile4_128x128>(g, stream);
    if (is(64, 128)) return launch_mx_linear<Tile4_64x128>(g, stream);
    return launch_mx_linear<Tile4_64x64>(g, stream);
  } else if constexpr (R == kRowsMx8) {
    if (is(256, 256)) return launch_mx_linear<Tile8_256x256>(g, stream);
    if (is(128, 256)) return launch_mx_linear<Tile8_128x256>(g, stream);
    if (is(128, 128)) return launch_mx_linear<Tile8_128x128>(g, stream);
    if (is(64, 128)) return launch_mx_linear<Tile8_64x128>(g, stream);
    return launch_mx_linear<Tile8_64x64>(g, stream);
  } else if constexpr (R == kRowsMx8Parts) {
    if (is(128, 128)) return launch_mx_linear<Tile8P_128x128>(g, stream);
    if (is(64, 128)) return launch_mx_linear<Tile8P_64x128>(g, stream);
    return launch_mx_linear<Tile8P_64x64>(g, stream);
  } else {
    const long long grid = linear_grid(&g, f.rows, f.cols);
    if (f.rows == 128) return launch_rows16<128, 1>(g, grid, stream);
    if (f.rows == 64) return launch_rows16<64, 1>(g, grid, stream);
    if (grid <= 2 * cus) return launch_rows16<32, 2>(g, grid, stream);
    return launch_rows16<32, 1>(g, grid, stream);
  }
}

// The checks of sizes.
static int check_sizes(int rows, int T, int K, int N) {
  if (T < 0 || K <= 0 || N <= 0) return LMOE_ERR_ARG;
  if (rows != kRowsBf16 && rows != kRowsMx8 && rows != kRowsMx4) return LMOE_ERR_UNSUPPORTED;
  return K % kMxGroup != 0 || N % 16 != 0 || K > kMxMaxColumns ? LMOE_ERR_SHAPE : LMOE_OK;
}
// 8-bit rows: what one instruction's fixed-point sums lose, some 1e-4 of a result, would be
// most of an f32 output's error and does not show beside a bf16 store's 1.7e-3.
static int rows_taken(int rows, int out_f32) { return rows == kRowsMx8 && out_f32 ? kRowsMx8Parts : rows; }

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_mx4_linear(const void* x, const void* x_scale, int rows, int T, int K, int N, const void* w,
                               const void* bias, int bias_f32, const void* add, void* out, int out_f32,
                               hipStream_t stream) {
  const int st = check_sizes(rows, T, K, N);
  if (st != LMOE_OK || T == 0) return st;
  if (x == nullptr || w == nullptr || out == nullptr || (x_scale == nullptr) != (rows == kRowsBf16)) return LMOE_ERR_ARG;
  if (misaligned16(x) || misaligned16(w) || misaligned16(bias) || misaligned16(add) || misaligned16(out))
    return LMOE_ERR_SHAPE;
  const size_t n = static_cast<size_t>(T) * K, wide = static_cast<size_t>(N);
  const Span o{out, T * wide * (out_f32 ? 4 : 2)};
  const Span in[5] = {{x, rows == kRowsBf16 ? 2 * n : rows == kRowsMx8 ? n : n / 2},
                      {x_scale, n / kMxGroup},
                      {w, wide / 16 * mx4_block_bytes(K)},
                      {bias, wide * (bias_f32 ? 4 : 2)},
                      {add, T * wide * 2}};
  for (int i = 0; i < 5; ++i)  // in place over add: each value is read where its sum is written
    if (overlap(o, in[i]) && !(i == 4 && add == out && !out_f32)) return LMOE_ERR_ARG;
  const LinearArgs g{x, static_cast<const uint8_t*>(x_scale), static_cast<const uint8_t*>(w), T, K, N, bias,
                     static_cast<const uint16_t*>(add), out, bias_f32 != 0, out_f32 != 0, 1};
  switch (rows_taken(rows, out_f32)) {
    case kRowsMx4: return launch_linear<kRowsMx4>(g, stream);
    case kRowsMx8: return launch_linear<kRowsMx8>(g, stream);
    case kRowsMx8Parts: return launch_linear<kRowsMx8Parts>(g, stream);
    default: return launch_linear<kRowsBf16>(g, stream);
  }
}

extern "C" int lmoe_mx4_linear_form(int rows, int out_f32, int T, int K, int N, int cus, int* form) {
  const int st = check_sizes(rows, T, K, N);
  if (st != LMOE_OK) return st;
  if (T == 0 || cus < 0 || form == nullptr) return LMOE_ERR_ARG;
  LinearArgs g{};
  g.T = T;
  g.K = K;
  g.N = N;
  const LinearForm f = linear_form(rows_taken(rows, out_f32), g, cus > 0 ? cus : device_cus());
  form[0] = f.rows;
  form[1] = f.cols;
  form[2] = f.split_k;
  return LMOE_OK;
}
