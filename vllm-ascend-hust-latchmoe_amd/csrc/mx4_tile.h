// Expert products over 4-bit weights in row tiles (prefill).
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

#include "mx4_few.h"

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

template <bool GU, bool A8, int BM, int CS>
__global__ __launch_bounds__(kTileWaves * 64, 2) void mx4_tile_kernel(Mx4Args g) {
  using C = Mx4Tile<A8, BM, CS>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int* s_pair = reinterpret_cast<int*>(smem + C::OFF_PAIR);
  uint32_t* s_scale = reinterpret_cast<uint32_t*>(smem + C::OFF_SCALE);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // work item: XCD-contiguous chunks of (row tile, column tile)
  constexpr int OUT_COLS = GU ? kTileCols / 2 : kTileCols;
  const int NT = (g.N + OUT_COLS - 1) / OUT_COLS;
  const SlotWindow win0 = load_window(g.tile_off, g.offsets, g.P, 0, lane);
  const SlotWindow win1 = load_window(g.tile_off, g.offsets, g.P, 64, lane);
  const int total = g.meta[LMOE_META_TILES] * NT;
  const int share = (total + 7) >> 3;
  const int jj = blockIdx.x >> 3;
  const int item = (blockIdx.x & 7) * share + jj;
  if (jj >= share || item >= total) return;
  const int tile = item / NT;
  const int n0 = (item - tile * NT) * OUT_COLS;
  const TileSlot ts = slot_of_tile(g.tile_off, g.offsets, g.P, tile, win0, win1, lane);
  const int slot = ts.slot;
  const int p0 = ts.p0 + (tile - ts.tile0) * BM;
  const int rows = min(BM, ts.p1 - p0);

  const int K = g.K;
  const int chunks = mx4_chunks(K);
  const int tail = K & (kMxChunk - 1);  // columns of a short last chunk, 0: none
  const size_t row_bytes = static_cast<size_t>(K) * (A8 ? 1 : 2);

  // this lane's source of each load instruction: row, and piece within a chunk
  auto a_row = [&](int q) { return (wave * C::QA + q) * C::RPL + lane / C::PIECES; };
  auto a_piece = [&](int q) { return (lane % C::PIECES) ^ C::sw(a_row(q)); };
  const char* a_src[C::QA];
#pragma unroll
  for (int q = 0; q < C::QA; ++q) {
    const int r = a_row(q);
    const int pos = p0 + (r < rows ? r : 0);
    const size_t src = GU ? g.sorted_pairs[pos] / g.topk : pos;
    a_src[q] = static_cast<const char*>(g.a) + src * row_bytes + a_piece(q) * 16;
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
    wsrc[j] = g.w + slot * g.w_slot_bytes + static_cast<size_t>(min(b0 + j, wblocks - 1)) * bb;
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
  for (int r = tid; r < BM; r += kTileWaves * 64) s_pair[r] = g.sorted_pairs[p0 + (r < rows ? r : 0)];
  if constexpr (A8) {
    const int groups = K / kMxGroup;
    const int r = tid & (BM - 1);  // a row's scales, some chunks of it
    const int pos = p0 + (r < rows ? r : 0);
    const uint8_t* sp = g.a_scale + static_cast<size_t>(GU ? g.sorted_pairs[pos] / g.topk : pos) * groups;
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
          RowFrag<true> x[2];
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
            for (int j = 0; j < 4; ++j) acc[i][j] = mx4_step<true>(w[j], sc[j], x[i & 1], acc[i][j]);
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
      store_act<A8>(g, p0 + r, n0 + 32 * wave, lane, r < rows, gate, up);
    } else {
      const int pair = s_pair[r];
      store_y(g, pair, n0 + 64 * wave, lane, r < rows, acc[i][0], acc[i][1]);
      if (b0 + 2 < wblocks) store_y(g, pair, n0 + 64 * wave + 32, lane, r < rows, acc[i][2], acc[i][3]);
    }
  }
}

}  // namespace lmoe
