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

// bf16 rows in row tiles: the shorter ones while they do not fill the card.  us of 128 / 64 /
// 32 rows (workgroups of 32 rows):
//   300 x 2048 x 5120   (200)   30.6 / 21.2 / 14.2
//   512 x 7168 x 7168   (448)   106 / 73.5 / 56.8
//   1024 x 7168 x 7168  (896)   108 / 94.0 / 108
//   4096 x 2048 x 5120  (2560)  79.3 / 71.1 / 86.8
//   4096 x 7168 x 7168  (3584)  316 / 321 / 381
static int rows16_height(const LinearArgs& g, int cus) {
  return tiles_of(g, 32, kTileCols) <= 2 * cus ? 32 : tiles_of(g, 64, kTileCols) <= 5 * cus ? 64 : 128;
}

// MX4 and MX8 rows: the shape with the least time by this measure, in tenths of a us: for
// each round of the workgroups that a CU has at once `round`, and for each of its chunks of K
// the time of 1, 2, .. of them (the last round may have fewer).
struct ShapeCost {
  int BM, BN, at_once, round;
  double chunk[4];
};
// MX4 rows, us of 256 x 256 / 128 x 128 / 64 x 128 / 64 x 64 tiles: 4096 x 7168 x 7168 118 /
// 146 / 184 / 252, 4096 x 2048 x 5120 39.9 / 35.2 / 39.6 / 46.5, 1024 x 7168 x 7168 51.0 /
// 45.4 / 55.9 / 63.5, 300 x 2048 x 5120 19.8 / 10.3 / 8.5 / 8.2, 300 x 1408 x 2048 15.5 / 8.8
// / 6.8 / 5.8
constexpr ShapeCost kShapes4[4] = {{256, 256, 1, 43, {8.3}}, {128, 128, 2, 0, {4.7, 6.5}},
                                   {64, 128, 3, 0, {3.4, 4.8, 6.6}}, {64, 64, 4, 0, {2.8, 3.6, 5.0, 6.4}}};
// MX8 rows, us of 256 x 256 / 128 x 256 / 128 x 128 / 64 x 128 / 64 x 64 tiles: 4096 x 7168 x
// 7168 161 / 182 / 198 / 243 / 436, 4096 x 2048 x 5120 54.3 / 51.5 / 46.8 / 54.7 / 67.4, 1024 x
// 7168 x 7168 73.2 / 46.0 / 55.1 / 64.8 / 78.9, 512 x 7168 x 7168 72.1 / 43.0 / 43.3 / 34.1 /
// 46.4, 300 x 2048 x 5120 25.7 / 16.1 / 13.1 / 9.0 / 9.2, 300 x 1408 x 2048 20.5 / 12.7 / 10.7 /
// 7.3 / 6.1
constexpr ShapeCost kShapes8[5] = {{256, 256, 1, 67, {12.0}}, {128, 256, 1, 41, {7.5}}, {128, 128, 2, 10, {7.5, 9.6}},
                                   {64, 128, 2, 25, {3.6, 5.5}}, {64, 64, 3, 15, {3.3, 4.2, 4.9}}};

// MX8 rows with f32 outputs, in two parts (twice the products; 256 x 256 tiles spill 112
// registers), us of 128 x 256 / 128 x 128 / 64 x 128 / 64 x 64 tiles: 4096 x 7168 x 7168 352 /
// 335 / 361 / 474, 4096 x 2048 x 5120 88.7 / 80.2 / 87.3 / 109, 1024 x 7168 x 7168 89.2 / 89.8 /
// 95.2 / 115, 512 x 7168 x 7168 85.0 / 63.3 / 52.5 / 64.8, 300 x 2048 x 5120 29.3 / 21.4 / 13.8 /
// 13.9, 300 x 1408 x 2048 21.8 / 16.3 / 10.4 / 8.4
constexpr ShapeCost kShapes8Parts[4] = {{128, 256, 1, 64, {14.0}}, {128, 128, 2, 48, {10.4, 15.2}},
                                        {64, 128, 2, 35, {6.2, 8.4}}, {64, 64, 3, 32, {4.3, 6.7, 8.0}}};

template <int S>
static LinearForm cheapest(const ShapeCost (&shapes)[S], const LinearArgs& g, int cus) {
  const int chunks = mx4_chunks(g.K);
  int best = 0;
  double least = 0;
  for (int s = 0; s < S; ++s) {
    const ShapeCost& c = shapes[s];
    const long long each = (tiles_of(g, c.BM, c.BN) + cus - 1) / cus;  // a CU's tiles
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
//              16 x 2048 x 5120   32 x 7168 x 7168      64 x 7168 x 7168      128 x 2048 x 5120
//   MX4 rows   4.4 4.7 5.0  -     15.3 12.2 15.8 19.0   27.0 20.6 15.2 19.5     -    -   9.3  6.8
//   MX8 rows    -   -   -   -       -    -    -    -    31.8 22.9 18.1 20.2   13.3 11.1 13.0  7.2
//   bf16 rows  5.4 6.4 7.3  -     20.8 15.2 23.5   -    37.0 25.8 23.2 44.3   15.3 12.5 15.6 13.8
// MX8 rows in two parts (f32 outputs) cost up to 0.4 us more there, 128 x 2048 x 5120 11.9 10.5
// 13.2 10.8, 64 x 7168 x 7168 31.3 22.1 17.8 27.1.
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
  return {rows16_height(g, cus), kTileCols, false};
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
    if (is(128, 256)) return launch_mx_linear<Tile8P_128x256>(g, stream);
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
