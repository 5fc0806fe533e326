// Products of MX rows (4 or 8 bits) with 4-bit weights in row tiles: the experts' products of
// MX4 rows, and the plain product of MX4 and MX8 rows.
//
// A workgroup of WR x WC waves computes BM rows by BN weight rows (gate-up: BN / 2 act
// columns, whose gate and up blocks alternate).  K goes by in chunks of 128, the depth of
// v_mfma_scale_f32_16x16x128; NB buffers of LDS hold a chunk of both operands each (a row's
// chunk is 64 bytes in 4 bits, 128 in 8; a 16-row block's 1 KiB, as it lies in the bank).
// Both go there from memory without passing through registers, NB - 1 chunks ahead, and are
// read by all waves that share them: with the weights in registers straight from memory, as
// few rows have them, 128 and 256 rows a wave spilled.
//
// In the middle of a chunk's products each wave waits for its loads of the next chunk and
// for the others; after that barrier the next chunk is in LDS and the buffer before this
// one's is free: loads for it are sent, and the last products run while the next chunk's
// first fragments come out of LDS.  So the matrix instructions never wait for a barrier with
// nothing to do.  No branch stands between them: past the last chunk the loads go on, out of
// range, which fetches nothing.
//
// LDS holds 16-byte piece p of row r at position p ^ sw(r), which puts the sixteen lanes of
// a read on different banks.  The scales of a quad (four chunks) are one dword for a lane's
// row and group on either side (byte c: chunk c), so the matrix instruction picks its bytes
// without any arithmetic.  The weights' scales lie that way in the bank; the rows' are put
// together from their 16 bytes a row.
//
// Bound: of 4-bit rows the plain product of 4096 x 7168 x 7168 takes 105 us (4.0 PFLOP/s; 20
// in a row 108 to 116 by the card's power; from registers 7.3 with random values, 9.7 with
// zeros).  With zeros, which cost no power, and 8192 columns, two full rounds of workgroups,
// 96: 8 us a round are its start and its stores (33 MB), a chunk takes 0.71 us where its
// products take 0.44, a chunk without loads and reads of LDS 0.65, without the barrier as well
// 0.58.  MX8 rows: 160 to 171 us (2.6 PFLOP/s; a large library product of 8-bit floats with
// one scale reaches 2.8), in two parts 341.  Four waves of 128 x 128 took 141 us to the 123 of
// this shape in the same run, six buffers with one workgroup a CU were slower.
//
// Every output adds its chunks in order, whatever the shape is: the same bits.
#pragma once

#include "mx4_tile.h"

namespace lmoe {

// n scales of a row from `at` on, from any address; past the row's groups, ones.
template <class T>
__device__ __forceinline__ T load_scales(const uint8_t* sp, int at, int groups) {
  T v;
  if (at + static_cast<int>(sizeof(T)) <= groups) {
    __builtin_memcpy(&v, sp + at, sizeof(T));
  } else {
    v = 0;
    for (int e = 0; e < static_cast<int>(sizeof(T)); ++e)
      v |= static_cast<T>(at + e < groups ? sp[at + e] : kScaleOne) << (8 * e);
  }
  return v;
}

// A lane's part of a 16 x 128 fragment of rows, from LDS; p: its row, sw: the row's.
template <int R>
struct TileFrag;
template <>
struct TileFrag<kRowsMx4> {
  i32x4_t v;
  __device__ __forceinline__ void read(const char* p, int lg, int sw) {
    v = *reinterpret_cast<const i32x4_t*>(p + ((lg ^ sw) * 16));
  }
  __device__ __forceinline__ i32x8_t operand() const { return __builtin_shufflevector(v, v, 0, 1, 2, 3, 0, 1, 2, 3); }
};
template <>
struct TileFrag<kRowsMx8> {
  i32x4_t lo, hi;
  __device__ __forceinline__ void read(const char* p, int lg, int sw) {
    lo = *reinterpret_cast<const i32x4_t*>(p + ((lg ^ sw) * 16));
    hi = *reinterpret_cast<const i32x4_t*>(p + (((4 + lg) ^ sw) * 16));
  }
  __device__ __forceinline__ i32x8_t operand() const { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
};

template <>
struct TileFrag<kRowsMx8Parts> : TileFrag<kRowsMx8> {};

// W x^T of one chunk; B: the byte of both scales.
template <int R, int B>
__device__ __forceinline__ f32x4_t mx_step(const i32x4_t w, int ws, const TileFrag<R>& x, int xs, f32x4_t acc) {
  const i32x8_t a = __builtin_shufflevector(w, w, 0, 1, 2, 3, 0, 1, 2, 3);
  if constexpr (R == kRowsMx8Parts) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, rows8_part<false>(x.operand()), acc, 4, 0, B, ws, B, xs);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, rows8_part<true>(x.operand()), acc, 4, 0, B, ws, B, xs);
  }
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, x.operand(), acc, 4 /* e2m1 */, R == kRowsMx8 ? 0 : 4, B, ws,
                                                          B, xs);
}

// A workgroup's shape: WR x WC waves of MI x NJ fragments of 16 rows by 16 weight rows, NB
// chunks of both operands in LDS.
template <int R_, int MI_, int NJ_, int WR_, int WC_, int NB_>
struct MxShape {
  static constexpr int R = R_, MI = MI_, NJ = NJ_, WR = WR_, WC = WC_, NB = NB_;
  static constexpr int BM = 16 * MI * WR, BN = 16 * NJ * WC;
  static constexpr int WAVES = WR * WC, THREADS = 64 * WAVES;
  static constexpr int PIECES = holds_mx8(R) ? 8 : 4;  // 16-byte pieces of a row's chunk
  static constexpr int ROWB = 16 * PIECES, RPL = 64 / PIECES;  // its bytes; rows of a load instruction
  static constexpr int PART_A = BM * ROWB, PART_B = BN * 64, STAGE = PART_A + PART_B;
  static constexpr int QA = PART_A / 1024 / WAVES, QB = BN / 16 / WAVES;  // load instructions of a wave and chunk
  static constexpr int OFF_SCALE = NB * STAGE;           // a quad's scales: BM x 16 bytes of rows,
  static constexpr int OFF_WSCALE = OFF_SCALE + BM * 16;  // BN / 16 blocks of 256 of weights
  static constexpr int OFF_PAIR = OFF_WSCALE + BN * 16;
  static constexpr int LDS = OFF_PAIR + BM * 4;
  static constexpr int PER_ROW = THREADS / BM;  // threads that bring a row's scales of a quad
  using scales_t = std::conditional_t<PER_ROW == 2, uint64_t, uint32_t>;
  static_assert(PER_ROW * sizeof(scales_t) == 16);
  static_assert(LDS <= 160 * 1024 && BM <= THREADS && QA * 1024 * WAVES == PART_A && QB * 16 * WAVES == BN);
  // piece p of row r lies at position p ^ sw(r)
  static __device__ __forceinline__ int sw(int r) {
    return holds_mx8(R) ? (r >> 1) & 7 : (0x78 >> (2 * ((r >> 2) & 3))) & 3;
  }
};

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// 16 (4) bytes a lane from base + lane_at + at to LDS, 1 KiB (256 bytes) from dst on,
// without passing through registers.  on: -1, or 0: the load is out of range and fetches
// nothing (its address is that of the first chunk or quad, inside the operand either way).
// ONCE: nobody reads them again.
template <bool ONCE>
__device__ __forceinline__ void buffer_to_lds16(const uint8_t* base, int on, char* dst, uint32_t lane_at, int at) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, __builtin_amdgcn_readfirstlane(on),
                                                   0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 16, lane_at, __builtin_amdgcn_readfirstlane(at & on), 0,
                                           ONCE ? 2 /* nt */ : 0);
}
__device__ __forceinline__ void buffer_to_lds4(const uint8_t* base, int on, char* dst, uint32_t lane_at, int at) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, __builtin_amdgcn_readfirstlane(on),
                                                   0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 4, lane_at, __builtin_amdgcn_readfirstlane(at & on), 0, 0);
}
// -1 where a < b, else 0; scalar arithmetic all the way
__device__ __forceinline__ int below(int a, int b) { return (a - b) >> 31; }

template <int N>
__device__ __forceinline__ void wait_vm_barrier() {
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <Op OP, class C>
__global__ __launch_bounds__(C::THREADS, 2) void mx_tile_kernel(TileArgs<OP> g) {
  constexpr bool GU = OP == Op::kGateUp, LIN = OP == Op::kLinear;
  constexpr int R = C::R, BM = C::BM, MI = C::MI, NJ = C::NJ, NB = C::NB;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int* s_pair = reinterpret_cast<int*>(smem + C::OFF_PAIR);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave / C::WC, wc = wave - wr * C::WC;
  const int K = g.K, N = g.N;

  constexpr int OUT_COLS = GU ? C::BN / 2 : C::BN;
  int slot = 0, p0, rows, n0;
  // Experts, low tiles: weights that one row tile reads are read once.  Fetched so, from the
  // loop on, they leave the caches to the rows (60 experts of 2048 x 1408, 22 rows each, none
  // in a cache before: gate-up 39.4 -> 36.0 us, down 23.1 -> 21.1; 32 of 7168 x 2048 91 -> 81
  // and 52 -> 47.4); those that two tiles read, so fetched, cost 15% more than they do now.
  // (The first chunks too: down 22.1.  The plain product gains nothing.)
  constexpr bool kOnce = !LIN && BM <= 64;
  bool alone = false;
  if constexpr (LIN) {
    if (!linear_tile(g, BM, OUT_COLS, &p0, &n0)) return;
    rows = min(BM, g.T - p0);
  } else {
    const SlotWindow win0 = load_window(g.tile_off, g.offsets, g.P, 0, lane);
    const SlotWindow win1 = load_window(g.tile_off, g.offsets, g.P, 64, lane);
    // work item: XCD-contiguous chunks of (row tile, column tile)
    const int NT = (N + OUT_COLS - 1) / OUT_COLS;
    const int total = g.meta[LMOE_META_TILES] * NT;
    const int share = (total + 7) >> 3;
    const int jj = blockIdx.x >> 3;
    const int item = (blockIdx.x & 7) * share + jj;
    if (jj >= share || item >= total) return;
    const int tile = __builtin_amdgcn_readfirstlane(item / NT);
    n0 = (item - tile * NT) * OUT_COLS;
    const TileSlot ts = slot_of_tile(g.tile_off, g.offsets, g.P, tile, win0, win1, lane);
    slot = ts.slot;
    p0 = ts.p0 + (tile - ts.tile0) * BM;
    rows = min(BM, ts.p1 - p0);
    alone = kOnce && __builtin_amdgcn_readfirstlane(ts.p1 - ts.p0) <= BM;
  }
  const int chunks = mx4_chunks(K);
  const int groups = K / kMxGroup;
  // the pair of the tile's row r; rows past the last repeat the first
  auto pair_of = [&](int r) -> int {
    if constexpr (LIN) return 0;
    else return g.sorted_pairs[p0 + (r < rows ? r : 0)];
  };
  // its row of the operand, from row0 on
  auto source_row = [&](int r, int pair) -> int {
    if constexpr (GU) return pair / g.topk;
    else return r < rows ? r : 0;
  };
  // rows: gate-up's lie anywhere, the others' from the tile's first on
  const size_t row0 = GU ? 0 : p0;
  const uint8_t* rows_base = uniform(static_cast<const uint8_t*>(g.a) + row_bytes<R>(row0, K));
  auto a_row = [&](int q) { return (wave * C::QA + q) * C::RPL + lane / C::PIECES; };
  auto a_piece = [&](int q) { return (lane % C::PIECES) ^ C::sw(a_row(q)); };
  int a_pair[C::QA];
#pragma unroll
  for (int q = 0; q < C::QA; ++q) a_pair[q] = GU ? pair_of(a_row(q)) : 0;
  const int s_row = tid / C::PER_ROW;  // the row whose scales this thread brings
  const int scale_pair = GU ? pair_of(s_row) : 0;
  const int my_pair = tid < BM ? pair_of(tid) : 0;
  asm volatile("" ::: "memory");  // on their way before the loads below, which do not need them
  // weight blocks; those past the matrix repeat the last one
  const int wblocks = (GU ? 2 * N : N) / 16;
  const int b0 = (GU ? 2 * n0 : n0) / 16;
  const int bb = mx4_block_bytes(K);
  const uint8_t* wbase = uniform(slot_weights(g, slot) + static_cast<size_t>(b0) * bb);
  const int last_block = wblocks - 1 - b0;
  // load q of chunk c's weights to buffer buf; past the last chunk the same loads, out of
  // range: they fetch nothing, and what they leave there is not read
  auto issue_w = [&](int q, int c, int buf, auto once) {
    const int at = (c >> 2) * kMxQuadBytes + 256 + (c & 3) * 1024;
    const int b = wave * C::QB + q;
    buffer_to_lds16<decltype(once)::value>(wbase, below(c, chunks), smem + buf * C::STAGE + C::PART_A + b * 1024,
                                           lane * 16, min(b, last_block) * bb + at);
  };
  uint32_t a_off[C::QA];
  const uint32_t tail = K - (chunks - 1) * kMxChunk;  // columns of the last chunk
  auto issue_a = [&](int q, int c, int buf) {
    // past the row's end, where the weights are zeros, columns of the chunk's first group
    // again: what is not a number there has made the row's sums so already
    const uint32_t piece = a_piece(q);
    const uint32_t back = piece * (128 / C::PIECES) >= tail ? piece * 16 & ~below(c + 1, chunks) : 0;
    // Experts: rows past the tile's last, whose sums are dropped, are not fetched (tiles of
    // 256, 4096 tokens x 8 of 128 experts, 2048 x 768: 95 -> 93 us, down 85 -> 81).  Products
    // of MX8 rows have no registers left for it, and one such tile a column.
    const int load = wave * C::QA + q;
    const int on = below(c, chunks) & (LIN ? -1 : below(load * C::RPL, rows));
    buffer_to_lds16<false>(rows_base, on, smem + buf * C::STAGE + load * 1024, a_off[q] - back, c * C::ROWB);
  };
  constexpr int LOADS = C::QA + C::QB;  // of a wave and chunk

  const int first = wc * NJ;  // this wave's weight blocks, from b0
  const bool wave_live = first <= last_block;
  const int quads = (chunks + 3) >> 2;
  auto issue_ws = [&](int q, int quad) {  // load q of a quad's weights' scales
    const int b = wave * C::QB + q;
    buffer_to_lds4(wbase, below(quad, quads), smem + C::OFF_WSCALE + b * 256, lane * 4,
                   min(b, last_block) * bb + quad * kMxQuadBytes);
  };
  // load n of a chunk
  auto issue = [&](int n, int c, int buf, auto once) {
    if (n < C::QA) issue_a(n, c, buf);
    else issue_w(n - C::QA, c, buf, once);
  };
  // Eight waves that send a chunk's loads all at once wait for each other's addresses (32
  // loads of 16 clocks each), so they send them between the products, FIRST of them behind
  // the barrier and the others before the next one: 4096 x 7168 x 7168 of MX4 rows 112 -> 108
  // us (of zeros, which cost no power, 100 -> 96), gate-up of 2049 tokens x 4 of 32 experts,
  // 7168 x 2048 185 -> 179, 1024 x 7168 x 7168 of MX8 rows 50.5 -> 48.  Two workgroups of four
  // waves a CU gain nothing, lower tiles lose (7168 x 2048 87 -> 94: the loads that go out
  // later arrive later), and with three buffers the later ones would not arrive in time.
  constexpr bool SPREAD = NB > 3 && C::WAVES == 8;
  constexpr int FIRST = SPREAD ? LOADS / 2 : LOADS;
#pragma unroll
  for (int q = 0; q < C::QB; ++q) issue_w(q, 0, 0, std::false_type{});
#pragma unroll
  for (int q = 0; q < C::QB; ++q) issue_ws(q, 0);
#pragma unroll
  for (int q = 0; q < C::QA; ++q)
    a_off[q] = static_cast<uint32_t>(source_row(a_row(q), a_pair[q])) * (holds_mx8(R) ? K : K >> 1) + a_piece(q) * 16;
  // the rows' scales of a quad, as they lie: PER_ROW threads to a row
  constexpr int SB = sizeof(typename C::scales_t);
  const uint8_t* my_scales = g.a_scale + (row0 + source_row(s_row, scale_pair)) * groups;
  typename C::scales_t qs;
  auto get_scales = [&](int quad) { qs = load_scales<typename C::scales_t>(my_scales, 16 * quad + tid % C::PER_ROW * SB, groups); };
  auto put_scales = [&]() { *reinterpret_cast<typename C::scales_t*>(smem + C::OFF_SCALE + tid * SB) = qs; };
  get_scales(0);
#pragma unroll
  for (int q = 0; q < C::QA; ++q) issue_a(q, 0, 0);
#pragma unroll
  for (int c = 1; c < NB - 1; ++c)
#pragma unroll
    for (int n = 0; n < (c == NB - 2 ? FIRST : LOADS); ++n) issue(n, c, c, std::false_type{});
  if constexpr (!LIN)
    if (tid < BM) s_pair[tid] = my_pair;
  put_scales();

  f32x4_t acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  const int fr = lane & 15;
  const int wrow = wr * 16 * MI;  // this wave's first row
  const int live = min(MI, max(0, (rows - wrow + 15) >> 4));
  // this lane's bytes of a fragment: rows from wrow on, weights from block `first` on
  const char* x_at = smem + (wrow + fr) * C::ROWB;
  const int fsw = C::sw(fr);  // fragments start at multiples of 16 rows
  const char* w_at = smem + C::PART_A + first * 1024 + lane * 16;
  const char* s_at = smem + C::OFF_SCALE + (wrow + fr) * 16;
  const char* ws_at = smem + C::OFF_WSCALE + first * 256 + lane * 4;
  const uint32_t pick = 0x0400u + 0x0101u * lg;  // byte lg of two dwords

  // NL: 16-row fragments computed, a compile-time count so that the products are
  // straight-line code; rows past the tile's last are dropped at the store
  auto main_loop = [&](auto nl_tag, auto once) __attribute__((always_inline)) {
    constexpr int NL = decltype(nl_tag)::value;
    constexpr int PAIRS = (NL + 1) / 2;
    int xs[NL > 0 ? NL : 1], ws[NJ];
    i32x4_t w[NJ];
    TileFrag<R> x[2][2];  // with a chunk's weights two fragments of rows; the next two are on their way
    int buf = 0;
    const char* xp = x_at;  // in the chunk's buffer
    auto read_w = [&](int j, const char* p) { w[j] = *reinterpret_cast<const i32x4_t*>(p + j * 1024); };
    auto read_x = [&](int to, int pair, const char* p) {
#pragma unroll
      for (int i = 2 * pair; i < 2 * pair + 2 && i < NL; ++i)
        x[to][i & 1].read(p + i * 16 * C::ROWB, lg, fsw);
    };
    // byte B of the scales: chunk c of its quad.  No branch: the products before the
    // barrier would sink behind it
    auto chunk = [&](int c, auto b_tag) __attribute__((always_inline)) {
      constexpr int B = decltype(b_tag)::value;
      const int before = buf == 0 ? NB - 1 : buf - 1, next = buf + 1 == NB ? 0 : buf + 1;
      // not a constant: past what an instruction's offset reaches each would get a register
      int next_at = next * C::STAGE;
      asm volatile("" : "+s"(next_at));
      const char *xn = x_at + next_at, *wn = w_at + next_at;
      // when every wave has got here chunk c + 1 is in LDS and chunk c - 1 read
      auto turn = [&]() {
        if constexpr (B == 2) {  // every wave has read this quad's scales
          put_scales();
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        wait_vm_barrier<(NB - 3) * LOADS + (B == 2 && NB > 3 ? C::QB : 0)>();  // scales behind chunk c + NB - 2
      };
      const int last = before == 0 ? NB - 1 : before - 1;
      constexpr int SENT = FIRST + (B == 1 ? C::QB : 0);
      auto send = [&](int n) {  // behind the barrier
        if (n < FIRST) issue(n, c + NB - 1, before, once);
        else issue_ws(n - FIRST, (c >> 2) + 1);
      };
      // before it: the rest of the chunk begun in the one before this
      auto send_rest = [&](int n) { issue(FIRST + n, c + NB - 2, last, once); };
      if constexpr (NL > 0) {
        // loads between the products, so that no wave waits for the others' addresses
        constexpr int BEFORE = PAIRS / 2 * NJ, AFTER = (PAIRS - PAIRS / 2) * NJ;  // groups of products
        constexpr int REST = LOADS - FIRST;
        if constexpr (BEFORE == 0)
#pragma unroll
          for (int n = 0; n < REST; ++n) send_rest(n);
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
          constexpr int first_x = B * PAIRS & 1;
          if (p == PAIRS / 2) {
            turn();
            if constexpr (!SPREAD)
#pragma unroll
              for (int n = 0; n < SENT; ++n) send(n);
          }
          if (p + 1 < PAIRS) read_x((first_x + p + 1) & 1, p + 1, xp);
          else read_x((first_x + p + 1) & 1, 0, xn);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int i = 2 * p; i < 2 * p + 2 && i < NL; ++i)
              acc[i][j] = mx_step<R, B>(w[j], ws[j], x[(first_x + p) & 1][i & 1], xs[i], acc[i][j]);
            if (p + 1 == PAIRS || SPREAD) __builtin_amdgcn_sched_barrier(0);
            if (p + 1 == PAIRS) read_w(j, wn);  // the next chunk's, as this one's are done with
            if constexpr (SPREAD) {
              const int k = p * NJ + j;
              if (k < BEFORE) {
#pragma unroll
                for (int n = k * REST / (BEFORE > 0 ? BEFORE : 1); n < (k + 1) * REST / (BEFORE > 0 ? BEFORE : 1); ++n)
                  send_rest(n);
              } else {
#pragma unroll
                for (int n = (k - BEFORE) * SENT / AFTER; n < (k - BEFORE + 1) * SENT / AFTER; ++n) send(n);
              }
            }
            if (p + 1 == PAIRS || SPREAD) __builtin_amdgcn_sched_barrier(0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int n = 0; n < LOADS - FIRST; ++n) send_rest(n);
        turn();
#pragma unroll
        for (int n = 0; n < SENT; ++n) send(n);
      }
      buf = next;
      xp = xn;
    };
    auto begin_quad = [&](int quad) __attribute__((always_inline)) {
      if constexpr (NL > 0) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) ws[j] = *reinterpret_cast<const int*>(ws_at + j * 256);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const i32x4_t v = *reinterpret_cast<const i32x4_t*>(s_at + i * 256);
          const uint32_t lo = __builtin_amdgcn_perm(v[1], v[0], pick), hi = __builtin_amdgcn_perm(v[3], v[2], pick);
          xs[i] = static_cast<int>(__builtin_amdgcn_perm(hi, lo, 0x05040100u));
        }
      }
      if (quad + 1 < quads) get_scales(quad + 1);
    };
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    wait_vm_barrier<(NB - 3) * LOADS + FIRST>();  // chunk 0 and the scales
    if constexpr (NL > 0) {
      read_x(0, 0, x_at);
#pragma unroll
      for (int j = 0; j < NJ; ++j) read_w(j, w_at);
    }
    int quad = 0;
    for (; quad < chunks >> 2; ++quad) {
      begin_quad(quad);
      chunk(4 * quad, std::integral_constant<int, 0>{});
      chunk(4 * quad + 1, std::integral_constant<int, 1>{});
      chunk(4 * quad + 2, std::integral_constant<int, 2>{});
      chunk(4 * quad + 3, std::integral_constant<int, 3>{});
    }
    const int rest = chunks & 3;
    if (rest > 0) {
      begin_quad(quad);
      chunk(4 * quad, std::integral_constant<int, 0>{});
      if (rest > 1) chunk(4 * quad + 1, std::integral_constant<int, 1>{});
      if (rest > 2) chunk(4 * quad + 2, std::integral_constant<int, 2>{});
    }
  };
  auto run = [&](auto once) __attribute__((always_inline)) {
    if (!wave_live || live == 0) main_loop(std::integral_constant<int, 0>{}, once);
    else if (MI > 6 && live > 6) main_loop(std::integral_constant<int, MI>{}, once);
    else if (MI > 4 && live > 4) main_loop(std::integral_constant<int, MI < 6 ? MI : 6>{}, once);
    else if (MI > 2 && live > 2) main_loop(std::integral_constant<int, MI < 4 ? MI : 4>{}, once);
    else if (MI > 1 && live > 1) main_loop(std::integral_constant<int, MI < 2 ? MI : 2>{}, once);
    else main_loop(std::integral_constant<int, 1>{}, once);
  };
  if (alone) run(std::integral_constant<bool, kOnce>{});
  else run(std::false_type{});
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load writes to LDS past the workgroup's end
  if (!wave_live) return;

#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int r = wrow + 16 * i + fr;
    if (i >= live) break;
#pragma unroll
    for (int j = 0; j < NJ; j += GU ? 4 : 2) {
      if (first + j > last_block) break;
      if constexpr (GU) {
        const f32x4_t gate[2] = {acc[i][j], acc[i][j + 2]}, up[2] = {acc[i][j + 1], acc[i][j + 3]};
        store_act<R>(g, p0 + r, n0 + 8 * (first + j), lane, r < rows, gate, up);
      } else if constexpr (LIN) {
        store_linear(g, p0 + r, n0 + 16 * (first + j), lane, r < rows, acc[i][j], acc[i][j + 1]);
      } else {
        store_y(g, s_pair[r], n0 + 16 * (first + j), lane, r < rows, acc[i][j], acc[i][j + 1]);
      }
    }
  }
}

// By rows and weight rows.
using Tile4_256x256 = MxShape<kRowsMx4, 8, 4, 2, 4, 4>;
using Tile4_128x256 = MxShape<kRowsMx4, 8, 4, 1, 4, 3>;
using Tile4_128x128 = MxShape<kRowsMx4, 4, 4, 2, 2, 4>;
using Tile4_64x128 = MxShape<kRowsMx4, 2, 4, 2, 2, 4>;
using Tile4_64x64 = MxShape<kRowsMx4, 2, 2, 2, 2, 4>;
using Tile8_256x256 = MxShape<kRowsMx8, 8, 4, 2, 4, 3>;
using Tile8_128x256 = MxShape<kRowsMx8, 4, 4, 2, 4, 4>;
using Tile8_128x128 = MxShape<kRowsMx8, 4, 4, 2, 2, 3>;
using Tile8_64x128 = MxShape<kRowsMx8, 2, 4, 2, 2, 4>;
using Tile8_64x64 = MxShape<kRowsMx8, 2, 2, 2, 2, 4>;
using Tile8P_128x128 = MxShape<kRowsMx8Parts, 4, 4, 2, 2, 3>;
using Tile8P_64x128 = MxShape<kRowsMx8Parts, 2, 4, 2, 2, 4>;
using Tile8P_64x64 = MxShape<kRowsMx8Parts, 2, 2, 2, 2, 4>;

template <Op OP, class C>
int launch_mx(const TileArgs<OP>& g, long long grid, hipStream_t stream) {
  if (grid > 0x7fffffffLL) return LMOE_ERR_SHAPE;
  static LdsRaised raised;
  const int st = raise_lds(reinterpret_cast<const void*>(mx_tile_kernel<OP, C>), raised);
  if (st != LMOE_OK) return st;
  mx_tile_kernel<OP, C><<<static_cast<unsigned>(grid), C::THREADS, C::LDS, stream>>>(g);
  LMOE_RETURN_LAUNCH();
}

// Experts: at most n_pairs / BM row tiles and a short one per slot.
template <bool GU, class C>
int launch_mx_experts(const Mx4Args& g, hipStream_t stream) {
  constexpr int cols = GU ? C::BN / 2 : C::BN;
  const long long tiles = g.n_pairs / C::BM + (g.n_pairs < g.P ? g.n_pairs : g.P);
  const long long blocks = tiles * ((g.N + cols - 1) / cols);
  return launch_mx<GU ? Op::kGateUp : Op::kDown, C>(g, 8 * ((blocks + 7) / 8), stream);
}

template <class C>
int launch_mx_linear(LinearArgs g, hipStream_t stream) {
  const long long grid = linear_grid(&g, C::BM, C::BN);
  return launch_mx<Op::kLinear, C>(g, grid, stream);
}

}  // namespace lmoe
