// Entry point of the product with one matrix of 4-bit weights.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "mx44_tile.h"
#include "mx4_linear.h"
#include "spans.h"

namespace lmoe {

template <int R, int RB, int NF, int NW>
static int launch_linear_few(const LinearArgs& g, hipStream_t stream) {
  const long long grid = (g.N / 16 + RB - 1) / RB * ((g.T + 16ll * NF - 1) / (16 * NF));
  if (grid > 0x7fffffffll) return LMOE_ERR_SHAPE;
  mx4_linear_few_kernel<R, RB, NF, NW><<<static_cast<unsigned>(grid), NW * 64, 0, stream>>>(g);
  LMOE_RETURN_LAUNCH();
}

template <int R>
static int launch_linear(const LinearArgs& g, hipStream_t stream) {
  if constexpr (R == kRowsMx4) {
    if (g.T > 512) return launch_mx44<Op::kLinear, Mx44Tile256>(Mx4Args{}, g, (g.T + 255ll) / 256, stream);
    if (g.T > 128) return launch_mx44<Op::kLinear, Mx44Tile128>(Mx4Args{}, g, (g.T + 127ll) / 128, stream);
    if (g.T > 32) return launch_mx44<Op::kLinear, Mx44Tile64>(Mx4Args{}, g, (g.T + 63ll) / 64, stream);
  }
  if (g.T <= 16) {
    if (g.N <= 16384) return launch_linear_few<R, 1, 1, 8>(g, stream);
    return launch_linear_few<R, 4, 1, 4>(g, stream);
  }
  return launch_linear_few<R, 4, 2, 4>(g, stream);
}

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_mx4_linear(const void* x, const void* x_scale, int rows, int T, int K, int N, const void* w,
                               const void* bias, int bias_f32, const void* add, void* out, int out_f32,
                               hipStream_t stream) {
  if (T < 0 || K <= 0 || N <= 0) return LMOE_ERR_ARG;
  if (rows != kRowsBf16 && rows != kRowsMx8 && rows != kRowsMx4) return LMOE_ERR_UNSUPPORTED;
  if (K % kMxGroup != 0 || N % 16 != 0) return LMOE_ERR_SHAPE;
  if (T == 0) return LMOE_OK;
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
                     static_cast<const uint16_t*>(add), out, bias_f32 != 0, out_f32 != 0};
  if (rows == kRowsMx4) return launch_linear<kRowsMx4>(g, stream);
  if (rows == kRowsMx8) return launch_linear<kRowsMx8>(g, stream);
  return launch_linear<kRowsBf16>(g, stream);
}
