// The norm in front of a MoE layer and 8-bit rows.
//
//   r = x + residual;  y = r / sqrt(mean(r^2) + eps) * weight
//
// r is formed and kept in f32: residual_out and both forms of y are rounded
// once, from it.  One workgroup per row, eight columns per thread and step, the
// row in registers between its two uses, so every byte is read and written
// once; what bounds it is HBM (a few operations per byte), and for one row the
// two dependent memory trips and the launch.  Measured: 4096 rows of 2048 columns, bf16
// residual, both forms of y, 12.7 us (76 MB at 6.0 TB/s); 1237 rows of 7168, f32
// residual, 24.5 us (116 MB at 4.7 TB/s, what a large copy reaches); one row 2.0 us.
// Rows to 8 bits alone, in a graph: 4096 rows of 2048 columns 5.8 us (25 MB at 4.4 TB/s,
// launch included), 4096 of 7168 15.5 us (89 MB at 5.7 TB/s), one row 2.4 to 3.2 us.
#include <hip/hip_runtime.h>

#include "mx.h"

namespace lmoe {

struct NormArgs {
  const uint16_t* x;
  const void* residual;    // bf16 or f32, null: none
  const void* weight;      // bf16 or f32, null: no norm (rows to 8 bits only)
  void* residual_out;
  uint16_t* out;           // null: not asked for
  uint8_t* q;              // null: not asked for
  uint8_t* scale;
  float eps;
  int H;
};

enum { kNone = 0, kBf16 = 1, kF32 = 2 };

__device__ __forceinline__ void unpack8(const uint4 v, float (&f)[8]) {
  f[0] = bf16lo(v.x); f[1] = bf16hi(v.x); f[2] = bf16lo(v.y); f[3] = bf16hi(v.y);
  f[4] = bf16lo(v.z); f[5] = bf16hi(v.z); f[6] = bf16lo(v.w); f[7] = bf16hi(v.w);
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}
template <int KIND>
__device__ __forceinline__ void load8(const void* p, size_t at, float (&f)[8]) {
  if constexpr (KIND == kF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 a = q[0], b = q[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    unpack8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at), f);
  }
}

// Eight columns to 8 bits.  Four neighbouring lanes hold a group of 32, which
// never straddles the end of the row (H % 32 == 0); the maximum over the four
// goes by two quad permutes.
__device__ __forceinline__ void store_mx8(const NormArgs& g, int row, int h, const float (&y)[8]) {
  uint32_t m = abs_bits(y[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) m = umax32(m, abs_bits(y[e]));
  m = umax32(m, dpp_u32<kDppQuadXor1>(m));
  m = umax32(m, dpp_u32<kDppQuadXor2>(m));
  const int b = mx8_scale_byte(__uint_as_float(m));
  const float s = mx_scale_f32(b);
  const uint2 v = make_uint2(pack_e4m3x4(y[0], y[1], y[2], y[3], s),
                             pack_e4m3x4(y[4], y[5], y[6], y[7], s));
  *reinterpret_cast<uint2*>(g.q + static_cast<size_t>(row) * g.H + h) = v;
  if ((h & (kMxGroup - 1)) == 0)
    g.scale[static_cast<size_t>(row) * (g.H / kMxGroup) + h / kMxGroup] = static_cast<uint8_t>(b);
}

// V steps of eight columns per thread hold the row.
template <int V, int RES, int WEIGHT>
__global__ __launch_bounds__(1024) void add_rms_norm_kernel(NormArgs g) {
  __shared__ float s_sum[16];
  const int row = blockIdx.x;
  const int H = g.H, step = blockDim.x * 8;
  const size_t base = static_cast<size_t>(row) * H;
  float r[V][8];
  float sum = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int h = v * step + threadIdx.x * 8;
    const bool in = h < H;
    load8<kBf16>(g.x, base + (in ? h : 0), r[v]);
    if constexpr (RES != kNone) {
      float a[8];
      load8<RES>(g.residual, base + (in ? h : 0), a);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[v][e] += a[e];
    }
    if (in) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += r[v][e] * r[v][e];
    }
  }
  if constexpr (RES != kNone) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int h = v * step + threadIdx.x * 8;
      if (h >= H) continue;
      if constexpr (RES == kF32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(g.residual_out) + base + h);
        p[0] = make_float4(r[v][0], r[v][1], r[v][2], r[v][3]);
        p[1] = make_float4(r[v][4], r[v][5], r[v][6], r[v][7]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(g.residual_out) + base + h) = pack8(r[v]);
      }
    }
  }
  if constexpr (WEIGHT != kNone) {
    sum = wave_sum(sum);
    const int nw = (blockDim.x + 63) >> 6;
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int w = 0; w < nw; ++w) sum += s_sum[w];
    const float inv = 1.0f / sqrtf(sum / static_cast<float>(H) + g.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int h = v * step + threadIdx.x * 8;
      float w[8];
      load8<WEIGHT>(g.weight, h < H ? h : 0, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[v][e] = r[v][e] * inv * w[e];
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int h = v * step + threadIdx.x * 8;
    if (h >= H) continue;
    if (g.out != nullptr) *reinterpret_cast<uint4*>(g.out + base + h) = pack8(r[v]);
    if (g.q != nullptr) store_mx8(g, row, h, r[v]);
  }
}

constexpr int kNormMaxCols = 4 * 1024 * 8;

template <int RES, int WEIGHT>
static void launch_norm(const NormArgs& g, int T, hipStream_t stream) {
  const int lanes = (g.H + 7) / 8;
  // as few steps per thread as 1024 threads allow, whole waves
  const int v = (lanes + 1023) / 1024;
  const int threads = ((lanes + v - 1) / v + 63) / 64 * 64;
  if (v == 1) add_rms_norm_kernel<1, RES, WEIGHT><<<T, threads, 0, stream>>>(g);
  else if (v == 2) add_rms_norm_kernel<2, RES, WEIGHT><<<T, threads, 0, stream>>>(g);
  else add_rms_norm_kernel<4, RES, WEIGHT><<<T, threads, 0, stream>>>(g);
}

static bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

struct Span {
  const void* p;
  size_t bytes;
};
static bool overlap(const Span& a, const Span& b) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.p), q = reinterpret_cast<uintptr_t>(b.p);
  return p != 0 && q != 0 && p < q + b.bytes && q < p + a.bytes;
}

// Whether an output would be written over another one, or over an input that other
// workgroups (weight: any) still read.  Only a row over itself is safe, where both
// start at one address and their rows are as long.
static bool clobbers(const NormArgs& g, int T, bool residual_f32, bool weight_f32) {
  const size_t n = static_cast<size_t>(T) * g.H;
  const size_t rb = residual_f32 ? 4 : 2;
  const Span in[3] = {{g.x, 2 * n}, {g.residual, rb * n}, {g.weight, static_cast<size_t>(g.H) * (weight_f32 ? 4 : 2)}};
  const Span out[4] = {{g.residual_out, rb * n}, {g.out, 2 * n}, {g.q, n}, {g.scale, n / kMxGroup}};
  const size_t in_row[3] = {2, rb, 0}, out_row[4] = {rb, 2, 1, 0};  // bytes of a column
  for (int o = 0; o < 4; ++o) {
    for (int i = 0; i < 3; ++i)
      if (overlap(out[o], in[i]) && !(out[o].p == in[i].p && out_row[o] == in_row[i] && in_row[i] != 0)) return true;
    for (int v = 0; v < o; ++v)
      if (overlap(out[o], out[v])) return true;
  }
  return false;
}

}  // namespace lmoe

using namespace lmoe;

extern "C" int lmoe_add_rms_norm(const void* x, int T, int H, const void* residual,
                                 int residual_f32, const void* weight, int weight_f32, float eps,
                                 void* residual_out, void* out, void* q, void* scale,
                                 hipStream_t stream) {
  if (T < 0 || H <= 0 || !(eps >= 0.0f)) return LMOE_ERR_ARG;
  if (H % 8 != 0 || H > kNormMaxCols) return LMOE_ERR_SHAPE;
  if (q != nullptr && H % kMxGroup != 0) return LMOE_ERR_SHAPE;
  if (T == 0) return LMOE_OK;
  if (x == nullptr || weight == nullptr || (out == nullptr && q == nullptr)) return LMOE_ERR_ARG;
  if ((residual == nullptr) != (residual_out == nullptr) || (q == nullptr) != (scale == nullptr))
    return LMOE_ERR_ARG;
  if (misaligned16(x) || misaligned16(residual) || misaligned16(weight) ||
      misaligned16(residual_out) || misaligned16(out) || misaligned16(q))
    return LMOE_ERR_SHAPE;
  const NormArgs g{static_cast<const uint16_t*>(x), residual, weight, residual_out,
                   static_cast<uint16_t*>(out), static_cast<uint8_t*>(q),
                   static_cast<uint8_t*>(scale), eps, H};
  if (clobbers(g, T, residual_f32 != 0, weight_f32 != 0)) return LMOE_ERR_ARG;
  if (residual == nullptr) {
    if (weight_f32) launch_norm<kNone, kF32>(g, T, stream);
    else launch_norm<kNone, kBf16>(g, T, stream);
  } else if (residual_f32) {
    if (weight_f32) launch_norm<kF32, kF32>(g, T, stream);
    else launch_norm<kF32, kBf16>(g, T, stream);
  } else {
    if (weight_f32) launch_norm<kBf16, kF32>(g, T, stream);
    else launch_norm<kBf16, kBf16>(g, T, stream);
  }
  LMOE_RETURN_LAUNCH();
}

extern "C" int lmoe_rows_to_mx8(const void* x, int T, int H, void* q, void* scale,
                                hipStream_t stream) {
  if (T < 0 || H <= 0) return LMOE_ERR_ARG;
  if (H % kMxGroup != 0 || H > kNormMaxCols) return LMOE_ERR_SHAPE;
  if (T == 0) return LMOE_OK;
  if (x == nullptr || q == nullptr || scale == nullptr) return LMOE_ERR_ARG;
  if (misaligned16(x) || misaligned16(q)) return LMOE_ERR_SHAPE;
  const NormArgs g{static_cast<const uint16_t*>(x), nullptr, nullptr, nullptr, nullptr,
                   static_cast<uint8_t*>(q), static_cast<uint8_t*>(scale), 0.0f, H};
  if (clobbers(g, T, false, false)) return LMOE_ERR_ARG;
  launch_norm<kNone, kNone>(g, T, stream);
  LMOE_RETURN_LAUNCH();
}
