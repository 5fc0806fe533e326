// Entry points of the expert products over 4-bit weights.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gemm_lds.h"
#include "mx4_few.h"
#include "mx4_tile.h"

LMOE_FLAGS_UNIT(mx4)

namespace lmoe {

// ---------------------------------------------------------------------------
// weighted combine of f32 rows by pair: out[t] = add[t] + sum_j w[t][j] y[t k + j],
// added in j order, one rounding.  A few tokens' rows come from L2; four columns
// per thread and one wave per workgroup spread them over the CUs (16 tokens x 8 rows of
// 2048: 3.8 us, of which the launch and two dependent loads are most).
// ---------------------------------------------------------------------------
constexpr int kCombineStep = 8;

template <bool SCAN>  // SCAN: which pairs have a slot is looked up from their ids
__global__ __launch_bounds__(64) void combine_f32_kernel(
    const float* __restrict__ y, const int32_t* __restrict__ row_idx, TokenIds o, int P, const uint16_t* __restrict__ w,
    int topk, int H, const uint16_t* __restrict__ add, uint16_t* __restrict__ out) {
  const int t = blockIdx.x;
  const int h = (blockIdx.y * 64 + threadIdx.x) * 4;
  if (h >= H) return;
  f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j0 = 0; j0 < topk; j0 += kCombineStep) {
    f32x4_t v[kCombineStep];
    float wj[kCombineStep];
    bool use[kCombineStep];
#pragma unroll
    for (int jj = 0; jj < kCombineStep; ++jj) {  // every load issued, masked rows dropped below
      const int j = j0 + jj;
      const bool in = j < topk;
      const int p = t * topk + (in ? j : 0);
      if constexpr (SCAN) use[jj] = in && slot_of_id(o, P, o.ids[p]) >= 0;
      else use[jj] = in && (row_idx == nullptr || row_idx[p] >= 0);
      if (in && !use[jj] && blockIdx.y == 0 && threadIdx.x == 0) add_device_flag(LMOE_FLAG_UNPLACED, 1);
      wj[jj] = bf16_to_f32(w[p]);
      v[jj] = *reinterpret_cast<const f32x4_t*>(y + static_cast<size_t>(p) * H + h);
    }
#pragma unroll
    for (int jj = 0; jj < kCombineStep; ++jj)
      if (use[jj]) acc += wj[jj] * v[jj];
  }
  if (add != nullptr) {
    const uint2 a = *reinterpret_cast<const uint2*>(add + static_cast<size_t>(t) * H + h);
    acc += f32x4_t{bf16lo(a.x), bf16hi(a.x), bf16lo(a.y), bf16hi(a.y)};
  }
  *reinterpret_cast<uint2*>(out + static_cast<size_t>(t) * H + h) =
      make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
}

static bool known_path(int path) {
  return path == LMOE_PATH_AUTO || path == LMOE_PATH_GEMV || path == LMOE_PATH_MFMA;
}
constexpr int kMaxSlots = 65535;  // a grid dimension

static bool bad16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

template <bool GU, bool SCAN>
static void launch_few(const Mx4Args& g, const TokenIds& o, hipStream_t stream) {
  constexpr int cols = kFewMxBlocks * (GU ? 8 : 16);
  const dim3 grid((g.N + cols - 1) / cols, SCAN || g.n_pairs < g.P ? g.n_pairs : g.P);
  if (g.a_scale != nullptr) mx4_few_kernel<GU, true, false, SCAN><<<grid, kFewMxWaves * 64, 0, stream>>>(g, o);
  else if (!GU && g.split) mx4_few_kernel<GU, false, !GU, SCAN><<<grid, kFewMxWaves * 64, 0, stream>>>(g, o);
  else if (GU || !SCAN) mx4_few_kernel<GU, false, false, GU && SCAN><<<grid, kFewMxWaves * 64, 0, stream>>>(g, o);
}

// Row tiles of BM rows, at most n_pairs / BM + one short one per slot.
constexpr int kFewTileBlocks = 512;  // two workgroups per CU: up to these, two chunks a stage

template <bool GU, bool A8, int BM, int CS>
static int launch_tiles(const Mx4Args& g, unsigned grid, hipStream_t stream) {
  const int lds = Mx4Tile<A8, BM, CS>::lds_bytes(mx4_chunks(g.K));
  static bool raised[64] = {};  // per device: dynamic LDS past 64 KiB allowed
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return static_cast<int>(e);
  if (dev < 0 || dev >= 64 || !raised[dev]) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(mx4_tile_kernel<GU, A8, BM, CS>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return static_cast<int>(e);
    if (dev >= 0 && dev < 64) raised[dev] = true;
  }
  mx4_tile_kernel<GU, A8, BM, CS><<<grid, kTileWaves * 64, lds, stream>>>(g);
  return LMOE_OK;
}

template <bool GU, bool A8, int BM>
static int launch_tiles(const Mx4Args& g, hipStream_t stream) {
  constexpr int cols = GU ? kTileCols / 2 : kTileCols;
  const long long tiles = g.n_pairs / BM + (g.n_pairs < g.P ? g.n_pairs : g.P);
  const long long blocks = tiles * ((g.N + cols - 1) / cols);
  const long long grid = 8 * ((blocks + 7) / 8);
  if (grid > 0x7fffffffLL) return LMOE_ERR_SHAPE;
  if constexpr (BM == 32) {
    if (blocks <= kFewTileBlocks) return launch_tiles<GU, A8, BM, 2>(g, static_cast<unsigned>(grid), stream);
  }
  return launch_tiles<GU, A8, BM, 1>(g, static_cast<unsigned>(grid), stream);
}

static bool known_block_m(int bm) { return bm == 32 || bm == 64 || bm == 128; }

// Whether rows of K columns fit the LDS of tiles of block_m rows (MX8 rows: their scales).
static bool tiles_fit(int block_m, bool a8, int K) {
  const int chunks = mx4_chunks(K);
  const int lds = block_m == 32   ? (a8 ? Mx4Tile<true, 32, 2>::lds_bytes(chunks) : Mx4Tile<false, 32, 2>::lds_bytes(chunks))
                  : block_m == 64 ? (a8 ? Mx4Tile<true, 64, 1>::lds_bytes(chunks) : Mx4Tile<false, 64, 1>::lds_bytes(chunks))
                                  : (a8 ? Mx4Tile<true, 128, 1>::lds_bytes(chunks) : Mx4Tile<false, 128, 1>::lds_bytes(chunks));
  return lds <= 160 * 1024;
}

template <bool GU, bool A8>
static int launch_tiles(const Mx4Args& g, int block_m, hipStream_t stream) {
  if (block_m == 32) return launch_tiles<GU, A8, 32>(g, stream);
  if (block_m == 64) return launch_tiles<GU, A8, 64>(g, stream);
  return launch_tiles<GU, A8, 128>(g, stream);
}

// path AUTO: row tiles past this many pairs per slot, on average, of bf16 and of MX8 rows
// (native.py has the figures)
constexpr int kFewPairsPerSlot[2] = {4, 6};

static bool many_pairs(bool a8, int n_pairs, int P) { return n_pairs > static_cast<long long>(kFewPairsPerSlot[a8]) * P; }

static bool takes_tiles(int path, int block_m, bool a8, int H, int I, int n_pairs, int P, bool split) {
  if (path != LMOE_PATH_AUTO) return path == LMOE_PATH_MFMA;
  return !split && known_block_m(block_m) && many_pairs(a8, n_pairs, P) && tiles_fit(block_m, a8, H) &&
         tiles_fit(block_m, a8, I);
}

// AUTO with a permutation built for other tiles (the bf16 kernels' 96, 256 or 320 rows):
// an error where row tiles are due, as with an explicit path.  The split-K kernel is
// right for any number of rows, but reads the weights once for every 32 of them.
static bool lacks_height(int path, int block_m, bool a8, int n_pairs, int P, bool split) {
  return path == LMOE_PATH_AUTO && !split && !known_block_m(block_m) && many_pairs(a8, n_pairs, P);
}

template <bool GU>
static int launch(const Mx4Args& g, int path, int block_m, hipStream_t stream) {
  if (lacks_height(path, block_m, g.a_scale != nullptr, g.n_pairs, g.P, g.split)) return LMOE_ERR_SHAPE;
  if (!takes_tiles(path, block_m, g.a_scale != nullptr, g.K, g.N, g.n_pairs, g.P, g.split)) {
    launch_few<GU, false>(g, TokenIds{}, stream);
  } else {
    if (g.split) return LMOE_ERR_UNSUPPORTED;
    if (!known_block_m(block_m) || !tiles_fit(block_m, g.a_scale != nullptr, g.K)) return LMOE_ERR_SHAPE;
    const int st = g.a_scale != nullptr ? launch_tiles<GU, true>(g, block_m, stream)
                                        : launch_tiles<GU, false>(g, block_m, stream);
    if (st != LMOE_OK) return st;
  }
  LMOE_RETURN_LAUNCH();
}

}  // namespace lmoe

using namespace lmoe;

extern "C" long long lmoe_mx4_bytes(int N, int K) {
  if (N <= 0 || K <= 0 || N % 16 != 0 || K % kMxGroup != 0) return -1;
  return static_cast<long long>(N / 16) * mx4_block_bytes(K);
}

extern "C" int lmoe_mx4_gateup_silu(const void* x, const void* x_scale, int T, int H, int I, int k,
                                    const void* w13_slots, int n_slots, const int32_t* offsets,
                                    const int32_t* sorted_pairs, const int32_t* active,
                                    const int32_t* tile_off, const int32_t* meta, int n_pairs,
                                    int block_m, int path, void* act, void* act_scale, int act_split,
                                    hipStream_t stream) {
  if (T < 0 || H <= 0 || I <= 0 || k <= 0 || n_slots <= 0 || n_pairs < 0) return LMOE_ERR_ARG;
  if (n_pairs != static_cast<long long>(T) * k) return LMOE_ERR_ARG;
  if (H % kMxGroup != 0 || I % kMxGroup != 0 || n_slots > kMaxSlots) return LMOE_ERR_SHAPE;
  if (!known_path(path)) return LMOE_ERR_UNSUPPORTED;
  if (n_pairs == 0) return LMOE_OK;
  if (x == nullptr || w13_slots == nullptr || offsets == nullptr || sorted_pairs == nullptr ||
      active == nullptr || tile_off == nullptr || meta == nullptr || act == nullptr)
    return LMOE_ERR_ARG;
  if ((x_scale == nullptr) != (act_scale == nullptr) || (act_scale != nullptr && act_split)) return LMOE_ERR_ARG;
  if (bad16(x) || bad16(w13_slots) || bad16(act)) return LMOE_ERR_SHAPE;
  const Mx4Args g{x, static_cast<const uint8_t*>(x_scale), static_cast<const uint8_t*>(w13_slots),
                  lmoe_mx4_bytes(2 * I, H), H, I, k, n_slots, n_pairs, offsets, sorted_pairs, active,
                  tile_off, meta, act, static_cast<uint8_t*>(act_scale), false, act_split != 0};
  return launch<true>(g, path, block_m, stream);
}

extern "C" int lmoe_mx4_down(const void* act, const void* act_scale, int act_split, int H, int I,
                             const void* w2_slots, int n_slots, const int32_t* offsets,
                             const int32_t* sorted_pairs, const int32_t* active,
                             const int32_t* tile_off, const int32_t* meta, int n_pairs, int block_m,
                             int path, void* y, int y_f32, hipStream_t stream) {
  if (H <= 0 || I <= 0 || n_slots <= 0 || n_pairs < 0) return LMOE_ERR_ARG;
  if (H % kMxGroup != 0 || I % kMxGroup != 0 || n_slots > kMaxSlots) return LMOE_ERR_SHAPE;
  if (!known_path(path)) return LMOE_ERR_UNSUPPORTED;
  if (n_pairs == 0) return LMOE_OK;
  if (act == nullptr || w2_slots == nullptr || offsets == nullptr || sorted_pairs == nullptr ||
      active == nullptr || tile_off == nullptr || meta == nullptr || y == nullptr || (act_scale != nullptr && act_split))
    return LMOE_ERR_ARG;
  if (bad16(act) || bad16(w2_slots) || bad16(y)) return LMOE_ERR_SHAPE;
  const Mx4Args g{act, static_cast<const uint8_t*>(act_scale), static_cast<const uint8_t*>(w2_slots),
                  lmoe_mx4_bytes(H, I), I, H, 1, n_slots, n_pairs, offsets, sorted_pairs, active,
                  tile_off, meta, y, nullptr, y_f32 != 0, act_split != 0};
  return launch<false>(g, path, block_m, stream);
}

extern "C" int lmoe_combine_f32(const void* y, const int32_t* row_idx, const uint16_t* w, int T, int k,
                                int H, const void* add, void* out, hipStream_t stream) {
  if (T < 0 || k <= 0 || H <= 0) return LMOE_ERR_ARG;
  if (H % 8 != 0) return LMOE_ERR_SHAPE;
  if (T == 0) return LMOE_OK;
  if (y == nullptr || w == nullptr || out == nullptr) return LMOE_ERR_ARG;
  if (bad16(y) || bad16(add) || bad16(out)) return LMOE_ERR_SHAPE;
  combine_f32_kernel<false><<<dim3(T, (H + 255) / 256), 64, 0, stream>>>(
      static_cast<const float*>(y), row_idx, TokenIds{}, 0, w, k, H, static_cast<const uint16_t*>(add),
      static_cast<uint16_t*>(out));
  LMOE_RETURN_LAUNCH();
}

// The layer of few or many tokens: what the four calls do, in one.
extern "C" int lmoe_mx4_fused_moe(const void* x, const void* x_scale, int T, int H, int I, int k,
                                  const void* w13_slots, const void* w2_slots, int n_slots,
                                  const uint16_t* w, const int32_t* ids, const int32_t* log2phy,
                                  int n_log2phy, int path, int block_m, const lmoe_mx4_workspace* ws,
                                  const void* add, void* out, hipStream_t stream) {
  if (ws == nullptr || T < 0 || k <= 0) return LMOE_ERR_ARG;
  const long long n = static_cast<long long>(T) * k;
  if (n > 0x7fffffffLL) return LMOE_ERR_SHAPE;
  if (T > 0 && (ids == nullptr || w == nullptr || out == nullptr)) return LMOE_ERR_ARG;
  // every check of the products before the permutation is queued
  if (H <= 0 || I <= 0 || n_slots <= 0) return LMOE_ERR_ARG;
  if (H % kMxGroup != 0 || I % kMxGroup != 0 || n_slots > kMaxSlots) return LMOE_ERR_SHAPE;
  if (!known_path(path)) return LMOE_ERR_UNSUPPORTED;
  if (T > 0) {
    if (x == nullptr || w13_slots == nullptr || w2_slots == nullptr || ws->act == nullptr || ws->y == nullptr ||
        (x_scale == nullptr) != (ws->act_scale == nullptr) || (x_scale != nullptr && ws->act_split))
      return LMOE_ERR_ARG;
    if (bad16(x) || bad16(w13_slots) || bad16(w2_slots) || bad16(ws->act) || bad16(ws->y) || bad16(add) || bad16(out))
      return LMOE_ERR_SHAPE;
    if (path == LMOE_PATH_MFMA && (!known_block_m(block_m) || !tiles_fit(block_m, x_scale != nullptr, H) ||
                                   !tiles_fit(block_m, x_scale != nullptr, I)))
      return LMOE_ERR_SHAPE;
    if (lacks_height(path, block_m, x_scale != nullptr, static_cast<int>(n), n_slots, false)) return LMOE_ERR_SHAPE;
  }
  const int split = ws->act_split && !takes_tiles(path, block_m, x_scale != nullptr, H, I, static_cast<int>(n), n_slots, false);
  int st = lmoe_permute(ids, static_cast<int>(n), log2phy, n_log2phy, n_slots, 0, block_m, ws->counts, ws->offsets,
                        ws->sorted_pairs, ws->row_idx, ws->active, ws->tile_off, ws->meta, ws->permute_workspace,
                        ws->permute_workspace_bytes, stream);
  if (st != LMOE_OK || T == 0) return st;
  st = lmoe_mx4_gateup_silu(x, x_scale, T, H, I, k, w13_slots, n_slots, ws->offsets, ws->sorted_pairs, ws->active,
                            ws->tile_off, ws->meta, static_cast<int>(n), block_m, path, ws->act, ws->act_scale, split,
                            stream);
  if (st != LMOE_OK) return st;
  st = lmoe_mx4_down(ws->act, ws->act_scale, split, H, I, w2_slots, n_slots, ws->offsets, ws->sorted_pairs, ws->active,
                     ws->tile_off, ws->meta, static_cast<int>(n), block_m, path, ws->y, ws->y_f32, stream);
  if (st != LMOE_OK) return st;
  return ws->y_f32 ? lmoe_combine_f32(ws->y, ws->row_idx, w, T, k, H, add, out, stream)
                   : lmoe_combine(ws->y, ws->row_idx, w, T, k, H, add, out, stream);
}

extern "C" int lmoe_mx4_decode_few(const void* x, const void* x_scale, int T, int H, int I, int k, const void* w13_slots,
                                   const void* w2_slots, int n_slots, const uint16_t* w, const int32_t* ids,
                                   const int32_t* log2phy, int n_log2phy, const void* add, void* act, void* act_scale,
                                   void* y, void* out, hipStream_t stream) {
  if (T < 0 || H <= 0 || I <= 0 || k <= 0 || n_slots <= 0 || n_log2phy < 0) return LMOE_ERR_ARG;
  if (H % kMxGroup != 0 || I % kMxGroup != 0 || n_slots > kMaxSlots || static_cast<long long>(T) * k > kScanMaxPairs)
    return LMOE_ERR_SHAPE;
  if (T == 0) return LMOE_OK;
  if (x == nullptr || w13_slots == nullptr || w2_slots == nullptr || w == nullptr || ids == nullptr || act == nullptr ||
      y == nullptr || out == nullptr || (x_scale == nullptr) != (act_scale == nullptr))
    return LMOE_ERR_ARG;
  if (bad16(x) || bad16(w13_slots) || bad16(w2_slots) || bad16(act) || bad16(y) || bad16(add) || bad16(out))
    return LMOE_ERR_SHAPE;
  const bool split = x_scale == nullptr;
  const TokenIds o{ids, log2phy, n_log2phy, nullptr, nullptr, 0, 0};
  const Mx4Args gu{x, static_cast<const uint8_t*>(x_scale), static_cast<const uint8_t*>(w13_slots),
                   lmoe_mx4_bytes(2 * I, H), H, I, k, n_slots, T * k, nullptr, nullptr, nullptr, nullptr, nullptr, act,
                   static_cast<uint8_t*>(act_scale), false, split};
  const Mx4Args dn{act, static_cast<const uint8_t*>(act_scale), static_cast<const uint8_t*>(w2_slots),
                   lmoe_mx4_bytes(H, I), I, H, 1, n_slots, T * k, nullptr, nullptr, nullptr, nullptr, nullptr, y, nullptr,
                   true, split};
  launch_few<true, true>(gu, o, stream);
  launch_few<false, true>(dn, o, stream);
  combine_f32_kernel<true><<<dim3(T, (H + 255) / 256), 64, 0, stream>>>(
      static_cast<const float*>(y), nullptr, o, n_slots, w, k, H, static_cast<const uint16_t*>(add),
      static_cast<uint16_t*>(out));
  LMOE_RETURN_LAUNCH();
}

extern "C" int lmoe_mx4_decode_one(const void* x, const void* x_scale, int H, int I, int k, const void* w13_slots,
                                   const void* w2_slots, int n_slots, const uint16_t* w, const int32_t* ids,
                                   const int32_t* log2phy, int n_log2phy, const void* w13_b,
                                   const void* w2_b, int n_slots_b, const int32_t* log2phy_b, int n_log2phy_b,
                                   const void* add, void* act, void* act_scale, void* out, hipStream_t stream) {
  if (H <= 0 || I <= 0 || k <= 0 || n_slots <= 0 || n_log2phy < 0) return LMOE_ERR_ARG;
  const bool two = w13_b != nullptr;
  if (two != (w2_b != nullptr) || two != (log2phy_b != nullptr) || n_slots_b < 0 || n_log2phy_b < 0) return LMOE_ERR_ARG;
  if (two && log2phy == nullptr) return LMOE_ERR_ARG;
  if (H % kMxGroup != 0 || I % kMxGroup != 0 || k > kMaxSlots) return LMOE_ERR_SHAPE;
  if (x == nullptr || w13_slots == nullptr || w2_slots == nullptr || w == nullptr || ids == nullptr ||
      act == nullptr || out == nullptr || (x_scale == nullptr) != (act_scale == nullptr))
    return LMOE_ERR_ARG;
  if (bad16(x) || bad16(w13_slots) || bad16(w2_slots) || bad16(act) || bad16(add) || bad16(out) ||
      bad16(w13_b) || bad16(w2_b))
    return LMOE_ERR_SHAPE;
  const TokenIds gate_up{ids, log2phy, n_log2phy, static_cast<const uint8_t*>(w13_b), log2phy_b, n_log2phy_b, n_slots_b};
  TokenIds down = gate_up;
  down.w_b = static_cast<const uint8_t*>(w2_b);
  const Mx4Args gu{x, static_cast<const uint8_t*>(x_scale), static_cast<const uint8_t*>(w13_slots),
                   lmoe_mx4_bytes(2 * I, H), H, I, k, n_slots, k, nullptr, nullptr, nullptr, nullptr, nullptr, act,
                   static_cast<uint8_t*>(act_scale), false, x_scale == nullptr};
  const Mx4Args dn{act, static_cast<const uint8_t*>(act_scale), static_cast<const uint8_t*>(w2_slots),
                   lmoe_mx4_bytes(H, I), I, H, 1, n_slots, k, nullptr, nullptr, nullptr, nullptr, nullptr, out, nullptr,
                   false, x_scale == nullptr};
  const dim3 grid(I / 32, k);
  const uint16_t* a = static_cast<const uint16_t*>(add);
  if (x_scale != nullptr) {
    mx4_one_gateup_kernel<true><<<grid, kOneMxWaves * 64, 0, stream>>>(gu, gate_up);
    mx4_one_down_kernel<true><<<H / 16, kOneMxWaves * 64, 0, stream>>>(dn, down, w, a);
  } else {
    mx4_one_gateup_kernel<false><<<grid, kOneMxWaves * 64, 0, stream>>>(gu, gate_up);
    mx4_one_down_kernel<false><<<H / 16, kOneMxWaves * 64, 0, stream>>>(dn, down, w, a);
  }
  LMOE_RETURN_LAUNCH();
}
