// Values to 4 bits (OCP MXFP4) and back: rows of activations, and weights in the form
// that the slot bank holds.
//
// A group of 32 neighbouring columns shares 2^e, e the smallest integer >= -127 with
// max |v| <= 6 * 2^e; each v / 2^e goes to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties
// to the even code.  Both steps are exact in f32 (a scale is a power of two), so the codes
// are those of the definition, whatever reads them.
//
// Everything here reads its input once and writes its output once; what bounds it is HBM.
// A lane takes eight neighbouring columns (one 16-byte load of bf16 values, one dword of
// codes), so that both sides of a wave's access are whole lines; four neighbouring lanes
// hold a group, and its maximum goes by two quad permutes.  Measured, there / back (a copy
// of 1 GiB here: 5.05 TB/s): rows 4096 x 7168 11.9 / 14.4 us, 4096 x 2048 3.8 / 6.4, one row
// 2.1 / 2.1 (an empty launch); banks of 128 x 1536 x 2048, each over and over, 184 / 176 us
// (5.5 / 5.8 TB/s), in turn 371 together, 32 x 4096 x 7168 431 / 427.
#include <hip/hip_runtime.h>

#include "mx.h"
#include "spans.h"

namespace lmoe {

// This lane's eight columns at p (columns).
template <bool F32>
__device__ __forceinline__ void load_columns(const void* p, size_t at, float (&v)[8]) {
  if constexpr (F32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 a = q[0], b = q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    v[0] = bf16lo(q.x); v[1] = bf16hi(q.x); v[2] = bf16lo(q.y); v[3] = bf16hi(q.y);
    v[4] = bf16lo(q.z); v[5] = bf16hi(q.z); v[6] = bf16lo(q.w); v[7] = bf16hi(q.w);
  }
}

// The scale byte of the group that this lane's quad of lanes holds.
__device__ __forceinline__ int group_scale_byte(const float (&v)[8]) {
  uint32_t m = abs_bits(v[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) m = umax32(m, abs_bits(v[e]));
  m = umax32(m, dpp_u32<kDppQuadXor1>(m));
  m = umax32(m, dpp_u32<kDppQuadXor2>(m));
  return mx4_scale_byte(__uint_as_float(m));
}

// 2^(byte - 127), also where it is no normal number; NaN for 255.
__device__ __forceinline__ float scale_value(int byte) {
  if (byte == 255) return __uint_as_float(0x7fc00000u);
  return byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(byte) << 23);
}

__device__ __forceinline__ float code_value(uint32_t code) {
  // +-0, .5: m / 2;  above, (1 + m / 2) 2^(x - 1)
  const uint32_t x = (code >> 1) & 3, m = code & 1;
  const float a = x == 0 ? 0.5f * static_cast<float>(m)
                         : __uint_as_float(((x + 126) << 23) | (m << 22));
  return code & 8 ? -a : a;
}

// Eight values of a dword of codes, stored in bf16 (exact: two mantissa bits) or f32.
template <bool F32>
__device__ __forceinline__ void store_values(void* out, size_t at, uint32_t word, float s) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = code_value(word >> (4 * e)) * s;
  if constexpr (F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
}

// ---------------------------------------------------------------------------
// rows: groups and their scales lie one after the other, whatever the row length is
// ---------------------------------------------------------------------------
constexpr int kQuantThreads = 256;
constexpr int kOctets = 2;  // of a lane, kQuantThreads apart, both on their way at once

template <bool F32>
__global__ __launch_bounds__(kQuantThreads) void rows_to_mx4_kernel(const void* __restrict__ x, size_t octets,
                                                                    uint32_t* __restrict__ q, uint8_t* __restrict__ scale) {
  const size_t first = static_cast<size_t>(blockIdx.x) * (kOctets * kQuantThreads) + threadIdx.x;
  float v[kOctets][8];
#pragma unroll
  for (int u = 0; u < kOctets; ++u) {
    const size_t o = first + u * kQuantThreads;
    load_columns<F32>(x, o < octets ? o * 8 : 0, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kOctets; ++u) {
    const size_t o = first + u * kQuantThreads;
    const int b = group_scale_byte(v[u]);
    if (o >= octets) break;  // groups are whole: so are quads of lanes
    q[o] = pack_e2m1x8(v[u], mx_scale_f32(b), b);
    if ((o & 3) == 0) scale[o >> 2] = static_cast<uint8_t>(b);
  }
}

template <bool F32>
__global__ __launch_bounds__(kQuantThreads) void mx4_rows_values_kernel(const uint32_t* __restrict__ q,
                                                                        const uint8_t* __restrict__ scale, size_t octets,
                                                                        void* __restrict__ out) {
  const size_t first = static_cast<size_t>(blockIdx.x) * (kOctets * kQuantThreads) + threadIdx.x;
  uint32_t word[kOctets];
  int b[kOctets];
#pragma unroll
  for (int u = 0; u < kOctets; ++u) {
    const size_t o = first + u * kQuantThreads, at = o < octets ? o : 0;
    word[u] = q[at];
    b[u] = scale[at >> 2];
  }
#pragma unroll
  for (int u = 0; u < kOctets; ++u) {
    const size_t o = first + u * kQuantThreads;
    if (o < octets) store_values<F32>(out, o * 8, word[u], scale_value(b[u]));
  }
}

// ---------------------------------------------------------------------------
// weights: a workgroup takes one quad (512 columns) of one block of 16 rows, each of its
// four waves four rows: the 16 lanes of a row have 128 columns, a chunk.  Codes go to the
// chunk's KiB (16 bytes of a group together, those of four rows side by side), the four
// chunks' scales of a row and group are one dword; the quad is put together in LDS and
// leaves in whole lines (straight from the lanes, a dword each, 128 x 1536 x 2048 took 222
// us to 186).
// ---------------------------------------------------------------------------
struct BankArgs {
  const void* w;     // [E, N, K], or the values to write
  uint8_t* bank;
  size_t units;      // quads of all blocks
  int N, K;
  bool gate_up;
};

struct BankUnit {
  uint8_t* quad;
  size_t row0;  // the matrix row of the block's first
  int k0;       // the quad's first column
  int chunks;   // of it, that the row has
};
__device__ __forceinline__ BankUnit bank_unit(const BankArgs& g, size_t unit) {
  const int quads = (g.K + 511) >> 9, blocks = g.N >> 4;
  const size_t block = unit / quads;  // of all experts
  const int q = static_cast<int>(unit - block * quads);
  const size_t expert = block / blocks;
  const int b = static_cast<int>(block - expert * blocks);
  // blocks of [gate; up] rows take turns
  const int row = g.gate_up ? (b & 1) * (g.N >> 1) + (b >> 1) * 16 : b * 16;
  const int left = mx4_chunks(g.K) - 4 * q;
  return {g.bank + block * mx4_block_bytes(g.K) + static_cast<size_t>(q) * kMxQuadBytes,
          expert * g.N + row, q << 9, left < 4 ? left : 4};
}

template <bool F32>
__global__ __launch_bounds__(kQuantThreads) void mx4_quantize_kernel(BankArgs g) {
  __shared__ __attribute__((aligned(16))) uint8_t s_quad[kMxQuadBytes];  // as the bank has it
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const BankUnit u = bank_unit(g, blockIdx.x);
  const int piece = lane & 15;  // eight columns of a chunk
  const int r = 4 * wave + (lane >> 4);
  const size_t base = (u.row0 + r) * static_cast<size_t>(g.K) + u.k0 + 8 * piece;
  const int at = r + 16 * (piece >> 2);  // the lane that a product gives this row and group to
  float v[4][8];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const bool in = u.k0 + c * kMxChunk + 8 * piece < g.K;
    load_columns<F32>(g.w, in ? base + c * kMxChunk : 0, v[c]);
    if (!in) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = 0.0f;
    }
  }
  uint32_t scales = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const bool in = u.k0 + c * kMxChunk + 8 * piece < g.K;  // the same for a group
    const int b = in ? group_scale_byte(v[c]) : kScaleOne;
    scales |= static_cast<uint32_t>(b) << (8 * c);
    *reinterpret_cast<uint32_t*>(s_quad + 256 + c * 1024 + at * 16 + 4 * (piece & 3)) = pack_e2m1x8(v[c], mx_scale_f32(b), b);
  }
  if ((piece & 3) == 0) *reinterpret_cast<uint32_t*>(s_quad + 4 * at) = scales;
  __syncthreads();
  if (wave == 0) *reinterpret_cast<uint32_t*>(u.quad + 4 * lane) = *reinterpret_cast<const uint32_t*>(s_quad + 4 * lane);
  if (wave < u.chunks)
    *reinterpret_cast<uint4*>(u.quad + 256 + wave * 1024 + 16 * lane) =
        *reinterpret_cast<const uint4*>(s_quad + 256 + wave * 1024 + 16 * lane);
}

template <bool F32>
__global__ __launch_bounds__(kQuantThreads) void mx4_bank_values_kernel(BankArgs g) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const BankUnit u = bank_unit(g, blockIdx.x);
  const int piece = lane & 15;
  const int r = 4 * wave + (lane >> 4);
  const size_t base = (u.row0 + r) * static_cast<size_t>(g.K) + u.k0 + 8 * piece;
  const int at = r + 16 * (piece >> 2);
  const uint32_t scales = *reinterpret_cast<const uint32_t*>(u.quad + 4 * at);
  uint32_t word[4];
#pragma unroll
  for (int c = 0; c < 4; ++c)
    word[c] = *reinterpret_cast<const uint32_t*>(u.quad + 256 + (c < u.chunks ? c : 0) * 1024 + at * 16 + 4 * (piece & 3));
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (u.k0 + c * kMxChunk + 8 * piece < g.K)
      store_values<F32>(const_cast<void*>(g.w), base + c * kMxChunk, word[c], scale_value((scales >> (8 * c)) & 255));
}

static unsigned grid_of(size_t n, size_t per) { return static_cast<unsigned>((n + per - 1) / per); }

// The checks of a bank call.
static int check_bank(const void* values, int E, int N, int K, int gate_up, const void* bank, int f32, BankArgs* g) {
  if (E < 0 || N <= 0 || K <= 0) return LMOE_ERR_ARG;
  if (N % 16 != 0 || K % kMxGroup != 0 || (gate_up && N % 64 != 0)) return LMOE_ERR_SHAPE;
  if (K > kMxMaxColumns) return LMOE_ERR_SHAPE;
  const size_t each = static_cast<size_t>(N / 16) * ((K + 511) / 512), units = E * each;
  if (each >= 0x7fffffffull || units >= 0x7fffffffull) return LMOE_ERR_SHAPE;
  if (E == 0) return LMOE_OK;
  if (values == nullptr || bank == nullptr) return LMOE_ERR_ARG;
  if (misaligned16(values) || misaligned16(bank)) return LMOE_ERR_SHAPE;
  const size_t n = static_cast<size_t>(E) * N;
  if (overlap({values, n * K * (f32 ? 4 : 2)}, {bank, n / 16 * mx4_block_bytes(K)})) return LMOE_ERR_ARG;
  *g = BankArgs{values, static_cast<uint8_t*>(const_cast<void*>(bank)), units, N, K, gate_up != 0};
  return LMOE_OK;
}

// The checks of a rows call.
static int check_rows(const void* values, int T, int H, const void* q, const void* scale, int f32) {
  if (T < 0 || H <= 0) return LMOE_ERR_ARG;
  const size_t n = static_cast<size_t>(T) * H;
  if (H % kMxGroup != 0 || n / 8 / (kOctets * kQuantThreads) >= 0x7fffffffull) return LMOE_ERR_SHAPE;
  if (T == 0) return LMOE_OK;
  if (values == nullptr || q == nullptr || scale == nullptr) return LMOE_ERR_ARG;
  if (misaligned16(values) || misaligned16(q)) return LMOE_ERR_SHAPE;
  const Span v{values, n * (f32 ? 4 : 2)}, c{q, n / 2}, s{scale, n / kMxGroup};
  return overlap(v, c) || overlap(v, s) || overlap(c, s) ? LMOE_ERR_ARG : LMOE_OK;
}

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_rows_to_mx4(const void* x, int x_f32, int T, int H, void* q, void* scale, hipStream_t stream) {
  const int st = check_rows(x, T, H, q, scale, x_f32);
  if (st != LMOE_OK || T == 0) return st;
  const size_t octets = static_cast<size_t>(T) * H / 8;
  const unsigned grid = grid_of(octets, kOctets * kQuantThreads);
  uint32_t* codes = static_cast<uint32_t*>(q);
  uint8_t* s = static_cast<uint8_t*>(scale);
  if (x_f32) rows_to_mx4_kernel<true><<<grid, kQuantThreads, 0, stream>>>(x, octets, codes, s);
  else rows_to_mx4_kernel<false><<<grid, kQuantThreads, 0, stream>>>(x, octets, codes, s);
  LMOE_RETURN_LAUNCH();
}

extern "C" int lmoe_mx4_rows_values(const void* q, const void* scale, int T, int H, void* out, int out_f32,
                                    hipStream_t stream) {
  const int st = check_rows(out, T, H, q, scale, out_f32);
  if (st != LMOE_OK || T == 0) return st;
  const size_t octets = static_cast<size_t>(T) * H / 8;
  const unsigned grid = grid_of(octets, kOctets * kQuantThreads);
  const uint32_t* codes = static_cast<const uint32_t*>(q);
  const uint8_t* s = static_cast<const uint8_t*>(scale);
  if (out_f32) mx4_rows_values_kernel<true><<<grid, kQuantThreads, 0, stream>>>(codes, s, octets, out);
  else mx4_rows_values_kernel<false><<<grid, kQuantThreads, 0, stream>>>(codes, s, octets, out);
  LMOE_RETURN_LAUNCH();
}

extern "C" int lmoe_mx4_quantize(const void* w, int w_f32, int E, int N, int K, int gate_up, void* bank,
                                 hipStream_t stream) {
  BankArgs g;
  const int st = check_bank(w, E, N, K, gate_up, bank, w_f32, &g);
  if (st != LMOE_OK || E == 0) return st;
  const unsigned grid = static_cast<unsigned>(g.units);
  if (w_f32) mx4_quantize_kernel<true><<<grid, kQuantThreads, 0, stream>>>(g);
  else mx4_quantize_kernel<false><<<grid, kQuantThreads, 0, stream>>>(g);
  LMOE_RETURN_LAUNCH();
}

extern "C" int lmoe_mx4_bank_values(const void* bank, int E, int N, int K, int gate_up, void* out, int out_f32,
                                    hipStream_t stream) {
  BankArgs g;
  const int st = check_bank(out, E, N, K, gate_up, bank, out_f32, &g);
  if (st != LMOE_OK || E == 0) return st;
  const unsigned grid = static_cast<unsigned>(g.units);
  if (out_f32) mx4_bank_values_kernel<true><<<grid, kQuantThreads, 0, stream>>>(g);
  else mx4_bank_values_kernel<false><<<grid, kQuantThreads, 0, stream>>>(g);
  LMOE_RETURN_LAUNCH();
}
