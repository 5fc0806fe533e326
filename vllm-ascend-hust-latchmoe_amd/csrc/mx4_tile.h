// Products of bf16 and MX8 rows with 4-bit weights in row tiles (prefill): the experts' two,
// and the plain product of bf16 rows.
//
// A workgroup of four waves computes BM rows of one slot by 256 weight rows:
// gate-up 128 act columns (gate and up), down 256 y columns.  Each wave takes all
// BM rows and 64 weight rows (four 16-row blocks; gate-up: gate, up, gate, up of
// 32 act columns).  Per stage, one or two chunks of 128 columns, the rows go to LDS
// without passing through registers (two buffers, the next stage in flight under this
// one's products), where all four waves read them; weights go from memory straight to
// registers, one stage ahead, since the bank's order is the fragments' order and no
// two waves share any.
//
// LDS holds 16-byte piece p of row r at position p ^ sw(r).  A 16-byte read goes
// by sixteen lanes at a time, 0-3, 12-15, 20-27 first and 4-11, 16-19, 28-31 next
// (and so from 32 on); lane l reads row l % 16 and a piece that steps with l / 16.
// sw = r / 2 for MX8 rows (8 pieces a chunk, two rows over all banks) and r + 4 for
// bf16 rows (16 pieces) puts each sixteen on sixteen different positions.  The e4m3
// scales of the whole tile are put into LDS once, by chunk and row.  (No bank
// conflicts are left of 6.5e6; that and weights loaded ahead took the gate-up product
// of 4096 tokens x 8 of 128 experts, 2048 x 768, from 187 to 126 us with MX8 rows.)
//
// What bounds it: in large prefills the matrix units and, between their bursts, the
// wait at each stage's barrier.  Those 32768 pairs, back to back, gate-up / down: bf16
// rows 195 / 118 us, 1.06 / 0.87 PFLOP/s (a large bf16 matrix product here: 1.33), the
// units 58% / 45% busy; MX8 rows 120 / 88 us, 1.72 / 1.17 PFLOP/s (a large e4m3 product: 2.93),
// 46% / 31% busy, the down product held by its 134 MB of y as well.  With few rows per
// slot it is the weights: 300 tokens 45 / 30 us, 214 / 117 MB at 4.7 / 3.9 TB/s.
// Measured and slower: 256-row tiles of eight waves (gate-up 230 us against 193),
// workgroups that stay for several tiles (220 against 200), two weight chunks ahead
// (the compiler then waits for every load), K in phases, raised wave priority,
// nontemporal weights (no gain; down slower).
//
// Every output adds its chunks in order, whatever BM is: the same bits.
#pragma once

#include <atomic>
#include <type_traits>

#include "mx4_linear.h"

namespace lmoe {

constexpr int kTileWaves = 4;
constexpr int kTileCols = 256;  // weight rows of a workgroup

__device__ __attribute__((aligned(16))) const uint32_t g_zero16[4] = {0, 0, 0, 0};

// CS: chunks of a stage.  Two where a stage's wait is what bounds it, on grids of few
// workgroups (gate-up us, one / two, 32 rows: 16 experts of 4096 x 1024, 128 tokens x 2,
// bf16 rows 34.2 / 25.1, MX8 rows 27.6 / 20.2; 16 of 2048 x 512 18.4 / 14.0; 8 of 4096 x
// 2048, 64 tokens x 2 27.9 / 19.9).  Where there are workgroups to fill a CU their number
// counts for more, and two chunks' registers cost it (64 tokens x 8 of 128 experts, 2048 x
// 768, 39.4 / 42.5; 61 x 4 of 60, 2048 x 1408, 34.2 / 36.3; 300 x 8 of 128 49.4 / 46.7).
template <bool A8, int BM_, int CS_>
struct Mx4Tile {
  static constexpr int BM = BM_;
  static constexpr int CS = CS_;
  static constexpr int NF = BM / 16;                 // 16-row fragments
  static constexpr int PIECES = A8 ? 8 : 16;         // 16-byte pieces of a row's chunk
  static constexpr int ROWB = PIECES * 16;
  static constexpr int PART = BM * ROWB;             // a chunk's rows
  static constexpr int STAGE = CS * PART;
  static constexpr int RPL = 64 / PIECES;            // rows one load instruction fills
  static constexpr int QA = PART / 1024 / kTileWaves;  // load instructions per wave and chunk
  static_assert(CS_ == 1 || BM_ < 64, "room for a stage's scales");
  static_assert(QA * kTileWaves * 1024 == PART, "whole load instructions");
  static constexpr int OFF_PAIR = 2 * STAGE;         // BM pair ids
  static constexpr int OFF_SCALE = OFF_PAIR + BM * 4;
  // scales go to LDS 64 dwords at a time: two chunks of 32 rows (two chunks a stage too)
  static constexpr int CHUNKS = BM < 64 ? 2 : 1;     // room for whole ones
  static int lds_bytes(int chunks) { return OFF_SCALE + (A8 ? BM * 4 * ((chunks + CHUNKS - 1) / CHUNKS * CHUNKS) : 0); }
  static __device__ __forceinline__ int sw(int r) { return A8 ? (r >> 1) & 7 : (r + 4) & 15; }
};

__device__ __forceinline__ void load_lds16b(const void* src, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
// every load of this wave has landed and its LDS accesses are done; then the others'
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The slot whose row tiles hold a tile, its first tile and its rows: the last slot
// whose tile_off is not past the tile (ascending; P + 1 entries).  A wave looks 64 of
// them up at once, one per lane, and has the first 128 on their way before it needs
// any: the start of a workgroup then waits for one load here.
struct SlotWindow {
  int t0, o0, o1;
};
__device__ __forceinline__ SlotWindow load_window(const int32_t* tile_off, const int32_t* offsets, int P, int first,
                                                  int lane) {
  const int at = min(first + lane, P - 1);
  return {tile_off[at], offsets[at], offsets[at + 1]};
}
struct TileSlot {
  int slot, tile0, p0, p1;
};
// v, next: the windows from 0 and from 64 on
__device__ __forceinline__ TileSlot slot_of_tile(const int32_t* tile_off, const int32_t* offsets, int P, int tile,
                                                 SlotWindow v, SlotWindow next, int lane) {
  for (int first = 0;; first += 64) {
    // lanes past the last slot repeat it; lane 0's entry is never past the tile
    const int last = min(63, P - 1 - first);
    const int k = min(__popcll(__ballot(v.t0 <= tile)) - 1, last);
    const bool here = k < 63 || first + 64 >= P || read_lane_i32(next.t0, 0) > tile;
    if (here) return {first + k, read_lane_i32(v.t0, k), read_lane_i32(v.o0, k), read_lane_i32(v.o1, k)};
    v = next;
    if (first + 128 < P) next = load_window(tile_off, offsets, P, first + 128, lane);
  }
}

__device__ __forceinline__ const uint8_t* slot_weights(const Mx4Args& g, int slot) { return g.w + slot * g.w_slot_bytes; }
__device__ __forceinline__ const uint8_t* slot_weights(const LinearArgs& g, int) { return g.w; }

// What a tile kernel computes: the experts' two products, or the product with one matrix
// (here bf16 rows', 8192 x 7168 x 7168 in 607 us, 1.39 PFLOP/s; a large library product 1.33).
enum class Op { kGateUp, kDown, kLinear };
template <Op OP>
using TileArgs = std::conditional_t<OP == Op::kLinear, LinearArgs, Mx4Args>;

// The tile of one workgroup of the plain product, its first row and column: false where
// there is none.  An XCD has a block of row tiles by column tiles, which shares its L2, and
// takes the row tiles of a column one after the other.
__device__ __forceinline__ bool linear_tile(const LinearArgs& g, int BM, int BN, int* p0, int* n0) {
  const int xcd = blockIdx.x & 7, jj = blockIdx.x >> 3;
  const int RT = (g.T + BM - 1) / BM, NT = (g.N + BN - 1) / BN, xcs = 8 / g.xcd_rows;
  const int xr = xcd / xcs, xc = xcd - xr * xcs;
  const int r0 = RT * xr / g.xcd_rows, rn = RT * (xr + 1) / g.xcd_rows - r0;
  const int c0 = NT * xc / xcs, cn = NT * (xc + 1) / xcs - c0;
  if (jj >= rn * cn) return false;
  const int col = __builtin_amdgcn_readfirstlane(jj / rn);
  *p0 = (r0 + jj - col * rn) * BM;
  *n0 = (c0 + col) * BN;
  return true;
}
// Its grid: the eight XCDs divide the row tiles by xcd_rows and the column tiles by the
// rest, as evenly as they can, then with the fewest bytes for each L2.
inline long long linear_grid(LinearArgs* g, long long BM, long long BN) {
  const long long RT = (g->T + BM - 1) / BM, NT = (g->N + BN - 1) / BN;
  if (RT > 0x7fffffffLL / 8 || NT > 0x7fffffffLL / 8) return 0x80000000LL;
  long long best = 0, best_lines = 0;
  for (int xr = 1; xr <= 8; xr *= 2) {
    const long long r = (RT + xr - 1) / xr, c = (NT * xr + 7) / 8;
    const long long items = r * c, lines = r * BM + c * BN;
    if (best == 0 || items < best || (items == best && lines < best_lines)) {
      best = items;
      best_lines = lines;
      g->xcd_rows = xr;
    }
  }
  return 8 * best;
}

template <Op OP, bool A8, int BM, int CS>
__global__ __launch_bounds__(kTileWaves * 64, 2) void mx4_tile_kernel(TileArgs<OP> g) {
  constexpr bool GU = OP == Op::kGateUp, LIN = OP == Op::kLinear;
  using C = Mx4Tile<A8, BM, CS>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int* s_pair = reinterpret_cast<int*>(smem + C::OFF_PAIR);
  uint32_t* s_scale = reinterpret_cast<uint32_t*>(smem + C::OFF_SCALE);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  constexpr int OUT_COLS = GU ? kTileCols / 2 : kTileCols;
  int slot = 0, p0, rows, n0;
  if constexpr (LIN) {
    if (!linear_tile(g, BM, OUT_COLS, &p0, &n0)) return;
    rows = min(BM, g.T - p0);
  } else {
    // work item: XCD-contiguous chunks of (row tile, column tile)
    const int NT = (g.N + OUT_COLS - 1) / OUT_COLS;
    const SlotWindow win0 = load_window(g.tile_off, g.offsets, g.P, 0, lane);
    const SlotWindow win1 = load_window(g.tile_off, g.offsets, g.P, 64, lane);
    const int total = g.meta[LMOE_META_TILES] * NT;
    const int share = (total + 7) >> 3;
    const int jj = blockIdx.x >> 3;
    const int item = (blockIdx.x & 7) * share + jj;
    if (jj >= share || item >= total) return;
    const int tile = item / NT;
    n0 = (item - tile * NT) * OUT_COLS;
    const TileSlot ts = slot_of_tile(g.tile_off, g.offsets, g.P, tile, win0, win1, lane);
    slot = ts.slot;
    p0 = ts.p0 + (tile - ts.tile0) * BM;
    rows = min(BM, ts.p1 - p0);
  }

  const int K = g.K;
  const int chunks = mx4_chunks(K);
  const int tail = K & (kMxChunk - 1);  // columns of a short last chunk, 0: none
  constexpr int R = A8 ? kRowsMx8 : kRowsBf16;

  auto source_row = [&](int pos) -> size_t {
    if constexpr (GU) return g.sorted_pairs[pos] / g.topk;
    else return pos;
  };
  // this lane's source of each load instruction: row, and piece within a chunk
  auto a_row = [&](int q) { return (wave * C::QA + q) * C::RPL + lane / C::PIECES; };
  auto a_piece = [&](int q) { return (lane % C::PIECES) ^ C::sw(a_row(q)); };
  const char* a_src[C::QA];
#pragma unroll
  for (int q = 0; q < C::QA; ++q) {
    const int r = a_row(q);
    const int pos = p0 + (r < rows ? r : 0);
    const size_t src = source_row(pos);
    a_src[q] = static_cast<const char*>(g.a) + row_bytes<R>(src, K) + a_piece(q) * 16;
  }
  const int stages = (chunks + CS - 1) / CS;
  auto issue = [&](int stage, int buf) {
#pragma unroll
    for (int e = 0; e < CS; ++e) {
      const int c = stage * CS + e;
      char* st = smem + buf * C::STAGE + e * C::PART + wave * C::QA * 1024;
      const int here = K - c * kMxChunk;  // columns of the chunk; past them, and in one past the last, zeros
      if (here >= kMxChunk) {
#pragma unroll
        for (int q = 0; q < C::QA; ++q) load_lds16b(a_src[q] + static_cast<size_t>(c) * C::ROWB, st + q * 1024);
      } else {
#pragma unroll
        for (int q = 0; q < C::QA; ++q) {
          const char* p = a_src[q] + static_cast<size_t>(c) * C::ROWB;
          if (a_piece(q) * (A8 ? 16 : 8) >= here) p = reinterpret_cast<const char*>(g_zero16);
          load_lds16b(p, st + q * 1024);
        }
      }
    }
  };

  // this wave's four weight blocks; blocks past the matrix repeat the last one
  const int wblocks = (GU ? 2 * g.N : g.N) / 16;
  const int b0 = (GU ? 2 * n0 : n0) / 16 + 4 * wave;
  const int bb = mx4_block_bytes(K);
  const bool wave_live = b0 < wblocks;
  const uint8_t* wsrc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    wsrc[j] = slot_weights(g, slot) + static_cast<size_t>(min(b0 + j, wblocks - 1)) * bb;
  const uint32_t code_at = lane * 16, scale_at = lane * 4;
  // codes of a stage's chunks (one past the last: the last's; its rows are zeros), and
  // the scales: byte c % 4 is chunk c's, of one dword for the whole stage
  auto load_w = [&](int stage, i32x4_t (&w)[CS][4], int (&sc)[4]) {
    typedef const __attribute__((address_space(1))) uint8_t* base_t;
    const int c0 = stage * CS;
    const int quad = (c0 >> 2) * kMxQuadBytes;
    uint32_t at = code_at, sat = scale_at;
    // up to 64 rows: the wave's base in scalar registers, the lane's offset (made here,
    // so that its 32 bits are seen) beside it: no address arithmetic.  Gate-up us, without
    // / with: 64 rows 55.1 / 52.5, 32 rows 47.2 / 45.7, but 128 rows 119.0 / 121.5.
    if constexpr (BM < 128) asm volatile("" : "+v"(at), "+v"(sat));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const base_t p = (base_t)(wsrc[j] + quad);
#pragma unroll
      for (int e = 0; e < CS; ++e) {
        const base_t codes = p + 256 + (min(c0 + e, chunks - 1) & 3) * 1024;
        w[e][j] = *(const __attribute__((address_space(1))) i32x4_t*)(codes + at);
      }
      sc[j] = *(const __attribute__((address_space(1))) int*)(p + sat);
    }
  };

  i32x4_t w_next[CS][4];
  int sc_next[4];
  issue(0, 0);
  load_w(0, w_next, sc_next);
  if constexpr (!LIN)
    for (int r = tid; r < BM; r += kTileWaves * 64) s_pair[r] = g.sorted_pairs[p0 + (r < rows ? r : 0)];
  if constexpr (A8) {
    const int groups = K / kMxGroup;
    const int r = tid & (BM - 1);  // a row's scales, some chunks of it
    const int pos = p0 + (r < rows ? r : 0);
    const uint8_t* sp = g.a_scale + source_row(pos) * groups;
    constexpr int STEP = kTileWaves * 64 / BM;
    if (tail == 0 && (reinterpret_cast<uintptr_t>(g.a_scale) & 3) == 0) {  // straight to LDS, 64 of them at a time
      for (int c = wave * 64 / BM; c < stages * CS; c += STEP) {
        const int mine = min(c + lane / BM, chunks - 1);  // two chunks where BM is 32
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)(sp + 4 * mine),
            (__attribute__((address_space(3))) void*)(s_scale + c * BM + (wave * 64 & (BM - 1))), 4, 0, 0);
      }
    } else {
      for (int c = tid / BM; c < stages * CS; c += STEP) {
        uint32_t v = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v |= static_cast<uint32_t>(4 * c + e < groups ? sp[e + 4 * c] : kScaleOne) << (8 * e);
        s_scale[c * BM + r] = v;
      }
    }
  }

  f32x4_t acc[C::NF][4];
#pragma unroll
  for (int i = 0; i < C::NF; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  const int fr = lane & 15;
  const int fsw = C::sw(fr);  // fragments start at multiples of 16 rows
  const int live = (rows + 15) >> 4;

  // NL: 16-row fragments computed, a compile-time count so that the products are
  // straight-line code; rows past the tile's last are dropped at the store
  auto main_loop = [&](auto nl_tag) {
    constexpr int NL = decltype(nl_tag)::value;
    for (int stage = 0; stage < stages; ++stage) {
      tile_barrier();  // the stage is in LDS; every wave is done with the other buffer
      i32x4_t wst[CS][4];
      int scst[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < CS; ++e) wst[e][j] = w_next[e][j];
        scst[j] = sc_next[j] >> (8 * (stage * CS & 3));
      }
      if (stage + 1 < stages) issue(stage + 1, (stage + 1) & 1);
      load_w(stage + 1 < stages ? stage + 1 : stage, w_next, sc_next);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < CS; ++e) {
        const int c = stage * CS + e;
        const i32x4_t(&w)[4] = wst[e];
        int sc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[j] = scst[j] >> (8 * e);
        const char* st = smem + (stage & 1) * C::STAGE + e * C::PART + fr * C::ROWB;
        // the next row fragment is on its way from LDS while this one is multiplied
        if constexpr (A8 && NL > 0) {
          RowFrag<kRowsMx8> x[2];
          const uint8_t* xs = reinterpret_cast<const uint8_t*>(s_scale + c * BM + fr) + lg;
          auto read = [&](int i) {
            const char* p = st + i * 16 * C::ROWB;
            const i32x4_t lo = *reinterpret_cast<const i32x4_t*>(p + ((lg ^ fsw) * 16));
            const i32x4_t hi = *reinterpret_cast<const i32x4_t*>(p + (((4 + lg) ^ fsw) * 16));
            x[i & 1].v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            x[i & 1].scale = xs[i * 64];
          };
          read(0);
#pragma unroll
          for (int i = 0; i < NL; ++i) {
            if (i + 1 < NL) read(i + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = mx4_step<kRowsMx8>(w[j], sc[j], x[i & 1], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
          }
        } else if constexpr (NL > 0) {
          float s[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) s[j] = mx_scale_f32(sc[j] & 255);
          bf16x8v_t x[2];
          auto read = [&](int n) {  // n: quarter of the chunk * NL + fragment
            const int k = n / NL, i = n % NL;
            x[n & 1] = *reinterpret_cast<const bf16x8v_t*>(st + i * 16 * C::ROWB + (((4 * lg + k) ^ fsw) * 16));
          };
          read(0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // quarters as mx4_step takes them
            bf16x8v_t wb[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) wb[j] = weights_bf16(w[j][k], s[j]);
#pragma unroll
            for (int i = 0; i < NL; ++i) {
              const int n = k * NL + i;
              if (n + 1 < 4 * NL) read(n + 1);
              __builtin_amdgcn_sched_barrier(0);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[j], x[n & 1], acc[i][j], 0, 0, 0);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
      }
    }
  };
  if (!wave_live) main_loop(std::integral_constant<int, 0>{});
  else if (C::NF > 4 && live > 6) main_loop(std::integral_constant<int, C::NF>{});
  else if (C::NF > 4 && live > 4) main_loop(std::integral_constant<int, C::NF < 6 ? C::NF : 6>{});
  else if (C::NF > 2 && live > 2) main_loop(std::integral_constant<int, C::NF < 4 ? C::NF : 4>{});
  else if (C::NF > 1 && live > 1) main_loop(std::integral_constant<int, C::NF < 2 ? C::NF : 2>{});
  else main_loop(std::integral_constant<int, 1>{});
  if (!wave_live) return;

#pragma unroll
  for (int i = 0; i < C::NF; ++i) {
    const int r = 16 * i + fr;
    if (i >= live) break;
    if constexpr (GU) {
      const f32x4_t gate[2] = {acc[i][0], acc[i][2]}, up[2] = {acc[i][1], acc[i][3]};
      store_act<R>(g, p0 + r, n0 + 32 * wave, lane, r < rows, gate, up);
    } else if constexpr (LIN) {
      store_linear(g, p0 + r, n0 + 64 * wave, lane, r < rows, acc[i][0], acc[i][1]);
      if (b0 + 2 < wblocks) store_linear(g, p0 + r, n0 + 64 * wave + 32, lane, r < rows, acc[i][2], acc[i][3]);
    } else {
      const int pair = s_pair[r];
      store_y(g, pair, n0 + 64 * wave, lane, r < rows, acc[i][0], acc[i][1]);
      if (b0 + 2 < wblocks) store_y(g, pair, n0 + 64 * wave + 32, lane, r < rows, acc[i][2], acc[i][3]);
    }
  }
}

// Devices on which a kernel may take all of LDS, which past 64 KiB it has to be allowed to.
// Host threads may call at once: each then asks for the same.
struct LdsRaised {
  std::atomic<bool> on[64] = {};
};
inline int raise_lds(const void* kernel, LdsRaised& raised) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return static_cast<int>(e);
  const bool known = dev >= 0 && dev < 64;
  if (known && raised.on[dev].load(std::memory_order_relaxed)) return LMOE_OK;
  e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  if (e != hipSuccess) return static_cast<int>(e);
  if (known) raised.on[dev].store(true, std::memory_order_relaxed);
  return LMOE_OK;
}

template <Op OP, bool A8, int BM, int CS>
int launch_tile(const TileArgs<OP>& g, long long grid, hipStream_t stream) {
  if (grid > 0x7fffffffLL) return LMOE_ERR_SHAPE;
  const int lds = Mx4Tile<A8, BM, CS>::lds_bytes(mx4_chunks(g.K));
  static LdsRaised raised;
  const int st = raise_lds(reinterpret_cast<const void*>(mx4_tile_kernel<OP, A8, BM, CS>), raised);
  if (st != LMOE_OK) return st;
  mx4_tile_kernel<OP, A8, BM, CS><<<static_cast<unsigned>(grid), kTileWaves * 64, lds, stream>>>(g);
  return LMOE_OK;
}

// Whether rows of K columns fit the LDS of tiles of block_m rows (MX8 rows: their scales;
// MX4 rows: whether the tiles' offsets reach them).
inline bool tiles_fit(int block_m, int rows, int K) {
  if (rows == kRowsMx4) return K <= kMxMaxColumns;
  const bool a8 = rows == kRowsMx8;
  const int chunks = mx4_chunks(K);
  const int lds = block_m == 32   ? (a8 ? Mx4Tile<true, 32, 2>::lds_bytes(chunks) : Mx4Tile<false, 32, 2>::lds_bytes(chunks))
                  : block_m == 64 ? (a8 ? Mx4Tile<true, 64, 1>::lds_bytes(chunks) : Mx4Tile<false, 64, 1>::lds_bytes(chunks))
                                  : (a8 ? Mx4Tile<true, 128, 1>::lds_bytes(chunks) : Mx4Tile<false, 128, 1>::lds_bytes(chunks));
  return lds <= 160 * 1024;
}

}  // namespace lmoe
