// The 8-bit linear over tiles of rows and columns, for many rows (see project.hip for the formula, project.h for the operands).
//
// Four wavefronts have a tile of y, each a quarter.  128 columns of K of the tile's rows and weights come by direct loads into one of two buffers in LDS, two steps
// ahead of the products and on into the workgroup's next tile, so that the loads of a tile's beginning run under the end of the one before it.  A load takes
// whole 128-byte lines of eight rows: with halves of lines of sixteen rows, which want no exchange in LDS, every line was fetched twice (8192 x 8192 x 8192: 655 us; this way 463).
// Nothing in a tile's end waits for memory of its own: scales and tables come by direct loads a tile ahead, the stores end under the next tile's first step (which took 16 us off 9392 rows, k 1024, n 8192, 8 slots of
// rank 64).  Measured in graph replay: 8192 x 8192 x 8192 493-510 us (2.2 PFLOP/s; the library's product with a scale a row and a column 480), 9392 rows, k 1024, n 8192 94-111 us as y's
// 154 MB fit the cache behind L2 or do not (library 106), with the adapters of 16 prompts 160-164, the matrix pipes busy for a third of this kernel's time.  What an adapters' step costs is less its products than what it
// finds out first and waits for.  Tiles of 256 x 128 with three buffers and eight wavefronts took 102 us for the base product where these took 95.  A word of every line of B asked for a tile ahead of the adapters' steps
// cost 1 us a tile more than it saved.
#include "common.h"
#include "dma.h"
#include "launch.h"
#include "lds.h"
#include "project.h"

#include <type_traits>

namespace mlora {

namespace {

constexpr int kXcds = 8;

// How the tiles of a call follow one another.  Workgroups go to the eight XCDs in turn; each XCD gets a run of tiles, in strips of eight row tiles (the last one of
// what is left), columns by columns, so that what works on an XCD at one time shares rows and columns in its L2.  The host divides: a tile's place takes no division.
struct Grid {
  int total, rows, columns;
  uint32_t strip_inverse, last_inverse;  // 2^32 over the tiles of a strip, and over the height of the last one, rounded down
};
constexpr int kStrip = 8;
struct Tile {
  int t, n;
};
__host__ __device__ __forceinline__ uint32_t inverse_of(uint32_t d) { return d > 1 ? static_cast<uint32_t>((1ull << 32) / d) : 0xffffffffu; }
__device__ __forceinline__ uint32_t divide(uint32_t v, uint32_t d, uint32_t inverse) {  // (the product is short of v / d by less than one)
  const uint32_t q = __umulhi(v, inverse);
  return v - q * d >= d ? q + 1 : q;
}
__device__ __forceinline__ Tile tile_of(const Grid& grid, int id) {
  const int share = grid.total / kXcds, more = grid.total % kXcds, xcd = id % kXcds;
  const uint32_t at = xcd * share + (xcd < more ? xcd : more) + id / kXcds;
  const uint32_t of_strip = kStrip * grid.columns, strip = divide(at, of_strip, grid.strip_inverse), in = at - strip * of_strip;
  const uint32_t high = grid.rows - strip * kStrip < kStrip ? grid.rows - strip * kStrip : kStrip;
  const uint32_t n = high == kStrip ? in / kStrip : divide(in, high, grid.last_inverse);
  return Tile{static_cast<int>(strip * kStrip + in - n * high), static_cast<int>(n)};
}

template <typename T, int TT, int NN, bool TAIL, int LORA> __global__ __launch_bounds__(256, LORA || TT * NN > 8 ? 2 : 3) void tiles8_kernel(MloraProjectArgs a, Grid grid) {
  constexpr int BT = 32 * TT, BN = 32 * NN, kStage = (BT + BN) * 128;
  extern __shared__ char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wt = wave >> 1, wn = wave & 1;
  const int total = grid.total;
  const uint32_t home = lds_address(lds);

  // the loads run two steps ahead of the products, over the tiles of this workgroup one behind the other
  int load_tile = blockIdx.x, load_k = 0, buffer = 0;
  bool loading = true;
  const char *x_from = nullptr, *w_from = nullptr;  // of the load that comes next
  uint32_t in_row[2];                               // where in its row a lane's piece lies, of rows 0 .. 7 and 8 .. 15 of sixteen
  uint32_t x_off[TT], w_off[NN];  // eight rows a load, whole lines of 128 bytes; a row's 16-byte pieces lie exchanged in LDS
  int load_t0 = 0, load_n0 = 0;

  // With adapters: rows in the order of their slots.  What a tile's rows are lies in LDS for four tiles, the one that is multiplied, those that are loaded and the one
  // behind them, which is asked for a tile ahead.
  const int32_t* const order = static_cast<const int32_t*>(a.workspace);
  struct Table {
    int32_t rows[BT], slots[BT], ends[BT];  // the last: where the row's slot ends
  };
  // The scales of the tiles' rows and columns likewise, by direct loads that come with a tile's first step.
  float* const scales = reinterpret_cast<float*>(lds + 2 * kStage);  // [4][BT + BN]
  Table* const tables = reinterpret_cast<Table*>(lds + 2 * kStage + 4 * (BT + BN) * 4);
  int turn = 0;
  auto load_table = [&](int id, int which) {  // (64 rows a wavefront; the last row stands for those behind it)
    const int at = (wave & 1) * 64 + lane;
    if ((wave & 1) * 64 >= BT) return;
    const int t = tile_of(grid, id < total ? id : total - 1).t * BT + at, within = t < a.num_rows ? t : a.num_rows - 1;
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(tables + (which & 3)) + (wave & 1) * 256);
    if (wave >> 1) {
      dma4v(order + 2 * a.num_rows + within, to + BT * 8);
    } else {
      dma4v(order + within, to);
      dma4v(order + a.num_rows + within, to + BT * 4);
    }
  };
  // The slices, one a lane.
  const int ranks = padded_ranks(a.r), width = a.num_slices * ranks;
  const bool beyond = LORA && *any_h_beyond(a);  // some row's h is an infinity or a NaN
  int slice_column = 0, slice_wide = 0, slice_b[2] = {0, 0};
  if constexpr (LORA == kStaged) {
    const int s = lane < a.num_slices ? lane : 0;
    slice_column = a.slices[s].y_col;
    slice_wide = lane < a.num_slices ? a.slices[s].n : 0;
    const uint64_t at = reinterpret_cast<uint64_t>(a.slices[s].b);
    slice_b[0] = static_cast<int>(at);
    slice_b[1] = static_cast<int>(at >> 32);
  }
  // The adapters' steps of a tile: its slots, for each the slices that its columns meet, of each 64 ranks at a time, of h one part after the other; of up to 32 ranks both parts at once, side by side.
  const bool narrow = ranks <= 32;
  struct Extra {
    int row, slot, stop, first, end, slice, c, part;  // the slot's first row in the tile (BT: no more) and where it stops, the slices
  };
  auto at_row = [&](const Table& table, Extra& e, int row) {
    e.row = row;
    if (row >= BT) return;
    const int slot = table.slots[row], stop = table.ends[row];
    e.slot = __builtin_amdgcn_readfirstlane(slot);
    e.stop = __builtin_amdgcn_readfirstlane(stop);
    if (e.slot < 0) e.row = BT;  // (rows without a slot come last)
  };
  auto first_extra = [&](const Table& table, int n0) {
    Extra e = {BT, -1, 0, 0, 0, 0, 0, 0};
    const unsigned long long meeting = __ballot(slice_wide && n0 + BN > slice_column && n0 < slice_column + slice_wide);
    if (!meeting) return e;
    e.first = e.slice = __builtin_ctzll(meeting);
    e.end = 64 - __builtin_clzll(meeting);
    at_row(table, e, 0);
    return e;
  };
  auto advance = [&](const Table& table, Extra& e, int t0) {
    if (!narrow && ++e.part < 2) return;
    e.part = 0;
    e.c += 64;
    if (e.c < ranks) return;
    e.c = 0;
    if (++e.slice < e.end) return;
    e.slice = e.first;
    at_row(table, e, e.stop < a.num_rows ? e.stop - t0 : BT);
  };
  Extra load_extra = {BT, -1, 0, 0, 0, 0, 0, 0}, coming = load_extra, current = load_extra;  // of the step that is loaded next, of the two that are multiplied in front of it
  // The column that row `at` of the weights' part of a step is, from the tile's first on.
  auto column_of = [&](int at) {
    const int block = at >> 4, f = block % NN, r = at & 15;
    return block / NN * (16 * NN) + 32 * (f >> 1) + 8 * (r >> 2) + 4 * (f & 1) + (r & 3);
  };
  // Piece c of a row's 128 bytes lies in LDS at c ^ (r / 2 % 8): sixteen rows' same piece, which a product reads at once, in all banks.  `bytes`: of a row; lanes behind its
  // end load its first ones, which are multiplied by zero.
  auto place = [&](uint32_t k, uint32_t bytes, bool ends) {
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      const uint32_t in = k + 16 * ((lane & 7) ^ (((lane >> 4) & 3) + 4 * odd));
      in_row[odd] = ends && in >= bytes ? 0 : in;
    }
  };
  int aimed = 0;  // tiles so far
  auto load_scales = [&]() {  // (the first half of the wavefronts has the rows, the other one the columns, 64 each; of smaller tiles not all have some)
    const int at = (wave & 1) * 64 + lane;
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(scales + (aimed & 3) * (BT + BN)) + (wave >> 1 ? BT * 4 : 0) + (wave & 1) * 256);
    if (wave >> 1) {
      if ((wave & 1) * 64 < BN) dma4v(a.w_scales + (load_n0 + at < a.n ? load_n0 + at : a.n - 1), to);
    } else if ((wave & 1) * 64 < BT) {
      int row;
      if constexpr (LORA != kNone) row = tables[(turn - 1) & 3].rows[at];
      else row = load_t0 + at < a.num_rows ? load_t0 + at : a.num_rows - 1;
      dma4v(a.x_scales + row, to);
    }
    ++aimed;
  };
  auto aim = [&]() {
    const Tile tile = tile_of(grid, load_tile);
    load_t0 = tile.t * BT;
    load_n0 = tile.n * BN;
    load_k = 0;
    place(0, a.k, TAIL);
    x_from = static_cast<const char*>(a.x) + (LORA ? 0 : static_cast<int64_t>(load_t0) * a.x_row);
    w_from = static_cast<const char*>(a.w) + static_cast<int64_t>(load_n0) * a.w_row;
    if constexpr (LORA) {
      const Table& table = tables[turn & 3];
#pragma unroll
      for (int i = 0; i < TT; ++i) x_off[i] = static_cast<uint32_t>(table.rows[(wave * TT + i) * 8 + (lane >> 3)]) * static_cast<uint32_t>(a.x_row);
      ++turn;
      load_table(load_tile + gridDim.x, turn);
    } else {
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const int row = (wave * TT + i) * 8 + (lane >> 3), most = a.num_rows - load_t0 - 1;
        x_off[i] = static_cast<uint32_t>((row < most ? row : most) * a.x_row);
      }
    }
#pragma unroll
    for (int i = 0; i < NN; ++i) {
      const int row = column_of((wave * NN + i) * 8 + (lane >> 3)), most = a.n - load_n0 - 1;
      w_off[i] = static_cast<uint32_t>((row < most ? row : most) * a.w_row);
    }
    load_scales();
  };
  // An adapters' step takes the rows' h for x, first one part of it and then the other, and the columns' B for w, which stays in registers for the second.
  auto aim_extra = [&]() {
    if (load_extra.part) {
      x_from += static_cast<int64_t>(a.num_rows) * width * 2;
      return;
    }
    const int wide = __builtin_amdgcn_readlane(slice_wide, load_extra.slice), column = __builtin_amdgcn_readlane(slice_column, load_extra.slice);
    const uint64_t b_of = static_cast<uint32_t>(__builtin_amdgcn_readlane(slice_b[0], load_extra.slice)) |
                          static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(slice_b[1], load_extra.slice))) << 32;
    x_from = reinterpret_cast<const char*>(intermediate(a) + static_cast<int64_t>(load_t0) * width + load_extra.slice * ranks);
    w_from = reinterpret_cast<const char*>(b_of) + static_cast<int64_t>(load_extra.slot) * wide * a.r * 2;
    // (narrow: the second four pieces of a row are the first four's ranks, of h's other part and of B once more)
    const uint32_t h_rest = static_cast<uint32_t>(a.num_rows) * static_cast<uint32_t>(width * 2);
    auto again = [&](int i) { return narrow && (((lane >> 2) ^ i) & 1); };
    if (narrow) {
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const uint32_t in = 16 * ((lane & 7) ^ (((lane >> 4) & 3) + 4 * odd));
        in_row[odd] = (in & 63) < static_cast<uint32_t>(ranks * 2) ? in : in & 64;
      }
    } else {
      place(load_extra.c * 2, ranks * 2, true);
    }
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int row = (wave * TT + i) * 8 + (lane >> 3), most = a.num_rows - load_t0 - 1;
      x_off[i] = static_cast<uint32_t>((row < most ? row : most) * width * 2) + (again(i) ? h_rest - 64 : 0);
    }
#pragma unroll
    for (int i = 0; i < NN; ++i) {
      const int in = load_n0 + column_of((wave * NN + i) * 8 + (lane >> 3)) - column;
      w_off[i] = static_cast<uint32_t>(in < 0 ? 0 : in < wide ? in : wide - 1) * static_cast<uint32_t>(a.r) * 2 - (again(i) ? 64 : 0);
    }
  };
  // What the next load takes, behind the one before it; between steps, since its branches would cut a step's code in pieces.
  auto prepare = [&]() {
    if constexpr (LORA == kStaged) {
      current = coming;
      coming = load_extra;
    }
    if (load_extra.row >= BT && load_k + 128 < a.k) {
      load_k += 128;
      if constexpr (TAIL) {
        place(load_k, a.k, true);
      } else {
        in_row[0] += 128;
        in_row[1] += 128;
      }
      return;
    }
    if constexpr (LORA == kStaged) {
      const Table& table = tables[(turn - 1) & 3];
      if (load_extra.row >= BT) load_extra = first_extra(table, load_n0);
      else advance(table, load_extra, load_t0);
      if (load_extra.row < BT) {
        aim_extra();
        return;
      }
    }
    load_tile += gridDim.x;
    loading = load_tile < total;
    if (loading) aim();
  };
  auto request = [&]() {
    if (!loading) return;
    const uint32_t to = __builtin_amdgcn_readfirstlane(home + buffer * kStage);
    const char *const x = uniform(x_from), *const w = uniform(w_from);
#pragma unroll
    for (int i = 0; i < TT; ++i) dma16_from(x, x_off[i] + in_row[i & 1], to + (wave * TT + i) * 1024);
    if (load_extra.row >= BT || !load_extra.part) {
#pragma unroll
      for (int i = 0; i < NN; ++i) dma16_from(w, w_off[i] + in_row[i & 1], to + (4 * TT + wave * NN + i) * 1024);
    }
    buffer ^= 1;
  };
  const char* const x_home = lds + wt * (TT * 2048) + m * 128;
  const char* const w_home = lds + (2 * TT + wn * NN) * 2048 + m * 128;
  const int piece[2] = {16 * (g ^ (m >> 1)), 16 * ((4 + g) ^ (m >> 1))};
  auto block_of = [&](const char* at, int i, Eight& to) {
#pragma unroll
    for (int p = 0; p < 2; ++p) to.piece[p] = *reinterpret_cast<const i32x4*>(at + i * 2048 + piece[p]);
  };

  f32x4 acc[TT][NN];
  int k = 0, now = 0;  // of the step that is multiplied
  // A step's first blocks into registers.
  auto begin = [&](Eight(&w)[NN], Eight(&x01)[2], int stage) {
#pragma unroll
    for (int n = 0; n < NN; ++n) block_of(w_home + stage, n, w[n]);
#pragma unroll
    for (int i = 0; i < 2; ++i) block_of(x_home + stage, i, x01[i]);
  };
  // Everything of this step has been read: its buffer takes the step after the next, which is there.
  bool stored = false;  // a whole tile's stores are younger than the loads of the step that has to be there: they need not have ended
  auto turn_over = [&]() {
    wait_lds();
    if (stored) wait_loads<TT * NN / 2>();
    else wait_loads<0>();
    stored = false;
    stage_barrier();
    request();
  };
  // (The last results may be read behind a branch that leaves a loop: the wait for a matrix instruction, which the next one would have to keep as well.)
  auto settle = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step of the base product: its blocks of w and the first two of x are in registers; leaves the next step's there.
  auto step = [&](Eight(&w)[NN], Eight(&x01)[2], Eight(&next_w)[NN], Eight(&next_x)[2]) {
    const char* const xs = x_home + now * kStage;
    Eight x[TT];
    x[0] = x01[0];
    x[1] = x01[1];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      if (t + 2 < TT) block_of(xs, t + 2, x[t + 2]);
      if (t == TT - 2) {
        turn_over();
        begin(next_w, next_x, (now ^ 1) * kStage);
      }
      if constexpr (TAIL) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (k + 64 * p + 16 * g >= a.k) x[t].piece[p] = i32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int n = 0; n < NN; ++n) acc[t][n] = mma8(w[n], x[t], acc[t][n]);
    }
    settle();
    k += 128;
    now ^= 1;
  };
  // A step of the adapters; leaves the next step's blocks where it found its own.
  int mine[TT];
  // What the lane's row of block t gains from a slot in one slice, one number at a time; where everything is NaN already, nothing.
  auto add_row = [&](int t, int slot, int s, int t0, int n0) {
    const int at = t0 + 16 * t + m < a.num_rows ? t0 + 16 * t + m : a.num_rows - 1;
    const uint16_t* const hi = intermediate(a) + static_cast<int64_t>(at) * width + s * ranks;
    const T* const b = static_cast<const T*>(a.slices[s].b) + static_cast<int64_t>(slot) * a.slices[s].n * a.r;
#pragma unroll
    for (int n = 0; n < NN; ++n) {
      f32x4 sum = acc[t][n];
      if (sum[0] != sum[0] && sum[1] != sum[1] && sum[2] != sum[2] && sum[3] != sum[3]) continue;
      add_slowly(b, a.slices[s].n, n0 + 32 * (n >> 1) + 4 * (n & 1) - a.slices[s].y_col, a.r, 0, a.r, hi, hi + static_cast<int64_t>(a.num_rows) * width, sum);
      acc[t][n] = sum;
    }
  };
  auto extra_step = [&](auto second, const Extra& e, int from, Eight(&w)[NN], Eight(&x01)[2]) {
    constexpr bool SECOND = decltype(second)::value;  // the second part of h: w is what the first one's step has made of it
    const char* const xs = x_home + now * kStage;
    Eight x[TT];
    x[0] = x01[0];
    x[1] = x01[1];
    auto rank_of = [&](const Extra& e, int p) { return e.c + (narrow ? 0 : 32 * p) + 8 * g; };
    if constexpr (!SECOND) {
      const int wide = __builtin_amdgcn_readlane(slice_wide, e.slice);
#pragma unroll
      for (int n = 0; n < NN; ++n) {  // (zero where there is no such rank or the column is none of the slice)
        const int in = from + 32 * (n >> 1) + 4 * (n & 1);
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (!(rank_of(e, p) < ranks && in >= 0 && in < wide)) w[n].piece[p] = i32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int t = 2; t < TT; ++t) block_of(xs, t, x[t]);
    // An infinity in B meets the leading part of h alone: with the other one, or its own second piece, it would make NaN.  Whether there is one a product with zeros shows: of numbers it is zero.
    f32x4 none[NN];
    if constexpr (!SECOND) {
      Pack8 zero;
      zero.raw = i32x4{0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int n = 0; n < NN; ++n) {
          Pack8 raw;
          raw.raw = w[n].piece[p];
          none[n] = Mma<T>::run(raw, zero, p ? none[n] : f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        }
    }
    turn_over();
    bool wild = false;
    if constexpr (!SECOND) {
      settle();
      f32x4 sum = none[0];
#pragma unroll
      for (int n = 1; n < NN; ++n) sum += none[n];
      wild = __ballot(!(sum[0] + sum[1] + sum[2] + sum[3] == 0.0f)) != 0;
    }
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int p = 0; p < 2; ++p)
        if (rank_of(e, p) >= ranks) x[t].piece[p] = i32x4{0, 0, 0, 0};
    auto finite = [&](const Pack8& hi, Pack8& of) {  // `of` where hi is a number, else zero
#pragma unroll
      for (int i = 0; i < 4; ++i) of.u[i] &= ~pair_mask(hi.u[i]);
    };
    auto keep_finite = [&](int p) {
#pragma unroll
      for (int n = 0; n < NN; ++n) {
        Pack8 b;
        b.raw = w[n].piece[p];
        finite(b, b);
        w[n].piece[p] = b.raw;
      }
    };
    [[maybe_unused]] Pack8 rest[NN][2];  // the second pieces of fp16's B
    if constexpr (BPiece<T>::kTwo) {
      if constexpr (!SECOND) {
#pragma unroll
        for (int n = 0; n < NN; ++n)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            Pack8 raw;
            raw.raw = w[n].piece[p];
            BPiece<T> b;
            b.from(raw);
            if (wild) finite(b.hi, b.lo);
            w[n].piece[p] = b.hi.raw;
            rest[n][p] = b.lo;
            if (narrow && p) rest[n][p].raw = i32x4{0, 0, 0, 0};
          }
      }
    }
    auto product = [&](int t, int n, f32x4 sum) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        Pack8 h, b;
        h.raw = x[t].piece[p];
        b.raw = w[n].piece[p];
        sum = Mma<__bf16>::run(b, h, sum);
        if constexpr (BPiece<T>::kTwo && !SECOND) sum = Mma<__bf16>::run(rest[n][p], h, sum);
      }
      return sum;
    };
    // (a lane's results are of one row, and come from that row's h alone: rows of other slots keep what they have, whatever is in this one's B)
    if (wild && narrow) keep_finite(1);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const bool own = mine[t] == e.slot;
      if (!__ballot(own)) continue;
#pragma unroll
        for (int n = 0; n < NN; ++n) {
          const f32x4 next = product(t, n, acc[t][n]);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][n][i] = own ? next[i] : acc[t][n][i];
        }
    }
    if (wild && !narrow) keep_finite(0), keep_finite(1);
    now ^= 1;
    if (SECOND || narrow) {
      begin(w, x01, now * kStage);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) block_of(x_home + now * kStage, i, x01[i]);
    }
  };

  if constexpr (LORA) {
    load_table(load_tile, 0);
    wait_loads<0>();
    stage_barrier();
  }
  aim();
  request();
  wait_lds();
  wait_loads<0>();
  stage_barrier();
  prepare();
  request();
  if (LORA != kNone && a.k <= 128) {  // (where that was the second tile's only step, the third one's table has to be there)
    wait_loads<0>();
    stage_barrier();
  }
  Eight w[2][NN], x01[2][2];
  begin(w[0], x01[0], 0);
  int done = 0;
  for (int id = blockIdx.x; id < total; id += gridDim.x, ++done) {
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int n = 0; n < NN; ++n) acc[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (k = 0; k < a.k;) {
      prepare();
      step(w[0], x01[0], w[1], x01[1]);
      if (k < a.k) {
        prepare();
        step(w[1], x01[1], w[0], x01[0]);
      } else {
#pragma unroll
        for (int n = 0; n < NN; ++n) w[0][n] = w[1][n];
#pragma unroll
        for (int i = 0; i < 2; ++i) x01[0][i] = x01[1][i];
      }
    }
    const Tile tile = tile_of(grid, id);
    const int t0 = tile.t * BT + wt * (16 * TT), n0 = tile.n * BN + wn * (16 * NN) + 8 * g;  // the lane's columns: n0 + 32 c + 0 .. 7
    const Table& table = tables[done & 3];
    const float* const scale = scales + (done & 3) * (BT + BN);
    {
      f32x4 columns[NN];
#pragma unroll
      for (int n = 0; n < NN; ++n) columns[n] = *reinterpret_cast<const f32x4*>(scale + BT + wn * (16 * NN) + 8 * g + 32 * (n >> 1) + 4 * (n & 1));
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int n = 0; n < NN; ++n) acc[t][n] *= columns[n];
    }
    // Rows whose h is not all numbers (bits of `odd`) are left out by the products, in which an infinity or a NaN would reach other targets' columns (B is zero there), and come last.
    unsigned odd = 0;
    if constexpr (LORA) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        mine[t] = table.slots[wt * (16 * TT) + 16 * t + m];
        if (!beyond || mine[t] < 0) continue;
        const int at = t0 + 16 * t + m < a.num_rows ? t0 + 16 * t + m : a.num_rows - 1;
        for (int j = 0; j < width; j += 8) {
          const i32x4 h = load128(intermediate(a) + static_cast<int64_t>(at) * width + j);
          if (pair_beyond(h[0]) || pair_beyond(h[1]) || pair_beyond(h[2]) || pair_beyond(h[3])) odd |= 1u << t;
        }
        if (odd >> t & 1) mine[t] = -1;
      }
    }
    if constexpr (LORA == kStaged) {
      while (coming.row < BT) {
        prepare();
        extra_step(std::false_type(), current, tile.n * BN + wn * (16 * NN) + 8 * (m >> 2) + (m & 3) - __builtin_amdgcn_readlane(slice_column, current.slice), w[0], x01[0]);
        if (narrow) continue;
        prepare();
        extra_step(std::true_type(), current, 0, w[0], x01[0]);
      }
      settle();
    }
    const bool whole = (tile.n + 1) * BN <= a.n && ((reinterpret_cast<uintptr_t>(a.y) | static_cast<uintptr_t>(a.y_row * 2)) & 15) == 0;
    if constexpr (LORA == kLoose) {  // every different slot among the wavefront's rows
      const uint16_t* const hi = intermediate(a);
      const uint16_t* const lo = hi + static_cast<int64_t>(a.num_rows) * width;
      const int begin = tile.n * BN + wn * (16 * NN);
      unsigned left[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) left[t] = static_cast<unsigned>(__ballot(mine[t] >= 0)) & 0xffffu;
      for (;;) {
        int slot = -1;
#pragma unroll
        for (int t = 0; t < TT; ++t)
          if (slot < 0 && left[t]) slot = __builtin_amdgcn_readlane(mine[t], __builtin_ctz(left[t]));
        if (slot < 0) break;
        unsigned has[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          has[t] = static_cast<unsigned>(__ballot(mine[t] == slot)) & 0xffffu;
          left[t] &= ~has[t];
        }
        for (int s = 0; s < a.num_slices; ++s) {
          const int wide = a.slices[s].n, column = a.slices[s].y_col;
          if (begin + 16 * NN <= column || begin >= column + wide) continue;
          const T* const b_slot = static_cast<const T*>(a.slices[s].b) + static_cast<int64_t>(slot) * wide * a.r;
          for (int c = 0; c < ranks; c += 32) {
            const int rank = c + 8 * g;
            const bool some = rank < ranks;
            Pack8 raw[NN], h[TT][2];
#pragma unroll
            for (int t = 0; t < TT; ++t) {
              // (places without a row or rank are read where there is one; of another slot's row nothing is kept)
              const int at = t0 + 16 * t + m < a.num_rows ? t0 + 16 * t + m : a.num_rows - 1;
              const int64_t from = static_cast<int64_t>(at) * width + s * ranks + (some ? rank : 0);
              h[t][0].raw = load128(hi + from);
              h[t][1].raw = load128(lo + from);
              if (!some) h[t][0].raw = h[t][1].raw = i32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int n = 0; n < NN; ++n) {
              const int in = begin + 32 * (n >> 1) + 8 * (m >> 2) + 4 * (n & 1) + (m & 3) - column;
              const bool there = some && in >= 0 && in < wide;
              const T* const from = b_slot + (there ? static_cast<int64_t>(in) * a.r + rank : 0);
              T* e = reinterpret_cast<T*>(&raw[n]);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                e[i] = from[there && rank + i < a.r ? i : 0];
                if (rank + i >= a.r) e[i] = static_cast<T>(0.0f);
              }
              if (!there) raw[n].raw = i32x4{0, 0, 0, 0};
            }
            BPiece<T> b[NN];
            Pack8 finite[NN];  // (an infinity in B meets the first part of h alone)
#pragma unroll
            for (int n = 0; n < NN; ++n) {
              b[n].from(raw[n]);
              finite[n] = b[n].hi;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t keep = ~pair_mask(finite[n].u[i]);
                finite[n].u[i] &= keep;
                if constexpr (BPiece<T>::kTwo) b[n].lo.u[i] &= keep;
              }
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
              if (!has[t]) continue;
              // (a lane's results are of one row, and come from that row's h alone: rows of other slots keep what they have, whatever is in this one's B)
              const bool own = mine[t] == slot;
#pragma unroll
              for (int n = 0; n < NN; ++n) {
                f32x4 next = Mma<__bf16>::run(b[n].hi, h[t][0], acc[t][n]);
                next = Mma<__bf16>::run(finite[n], h[t][1], next);
                if constexpr (BPiece<T>::kTwo) next = Mma<__bf16>::run(b[n].lo, h[t][0], next);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][n][i] = own ? next[i] : acc[t][n][i];
              }
            }
          }
        }
      }
    }

    if (LORA && __ballot(odd != 0)) {
#pragma unroll
      for (int t = 0; t < TT; ++t)
        if (odd >> t & 1)
          for (int s = 0; s < a.num_slices; ++s) add_row(t, table.slots[wt * (16 * TT) + 16 * t + m], s, t0, n0);
    }

    float bias[NN / 2][8];
#pragma unroll
    for (int c = 0; c < NN / 2; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) bias[c][i] = a.bias ? to_f32(static_cast<const T*>(a.bias)[n0 + 32 * c + i < a.n ? n0 + 32 * c + i : a.n - 1]) : 0.0f;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int at = t0 + 16 * t + m;
      if (at >= a.num_rows) continue;
      const int row = LORA ? table.rows[wt * (16 * TT) + 16 * t + m] : at;
      const float of_row = scale[wt * (16 * TT) + 16 * t + m];
      T* const y = static_cast<T*>(a.y) + static_cast<int64_t>(row) * a.y_row + n0;
#pragma unroll
      for (int c = 0; c < NN / 2; ++c) {
        T out[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = from_f32<T>(__builtin_fmaf(acc[t][2 * c + i / 4][i % 4], of_row, bias[c][i]));
        if (whole) {
          i32x4 word;
          __builtin_memcpy(&word, out, 16);
          store128(y + 32 * c, word);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n0 + 32 * c + i < a.n) y[32 * c + i] = out[i];
        }
      }
    }
    // Tiles of one step run three ahead of a wavefront that is still here: the table that is asked for next is the one that it reads.  (Of two steps and more the loads are two tiles ahead at most.)
    if (LORA != kNone && a.k <= 128) {
      wait_lds();
      stage_barrier();
    }
    stored = whole && (tile.t + 1) * BT <= a.num_rows && (LORA == kNone || a.k > 128);  // (of tiles of one step the next table comes behind the stores and has to be there)
  }
}

template <typename T, int TT, int NN, bool TAIL, int LORA> void launch(const MloraProjectArgs* a) {
  constexpr auto kernel = tiles8_kernel<T, TT, NN, TAIL, LORA>;
  constexpr int bytes = 2 * (32 * TT + 32 * NN) * 128 + 4 * (32 * TT + 32 * NN) * 4 + (LORA ? 4 * 3 * 32 * TT * 4 : 0);
  allow_lds<kernel>(bytes);
  Grid grid = {};
  grid.rows = (a->num_rows + 32 * TT - 1) / (32 * TT);
  grid.columns = (a->n + 32 * NN - 1) / (32 * NN);
  grid.total = grid.rows * grid.columns;
  grid.strip_inverse = inverse_of(kStrip * grid.columns);
  grid.last_inverse = inverse_of(grid.rows % kStrip);
  const int most = 256 * (TT * NN > 8 ? 2 : TT * NN > 4 ? 3 : 4);
  kernel<<<grid.total < most ? grid.total : most, 256, bytes, static_cast<hipStream_t>(a->stream)>>>(*a, grid);
}
template <typename T, int TT, int NN, int LORA> void launch_k(const MloraProjectArgs* a) {
  if (a->k % 128) launch<T, TT, NN, true, LORA>(a);
  else launch<T, TT, NN, false, LORA>(a);
}
template <typename T, int TT, int NN> void launch_lora(const MloraProjectArgs* a) {
  if (a->num_slices) launch_k<T, TT, NN, kStaged>(a);
  else launch_k<T, TT, NN, kNone>(a);
}
template <typename T> void launch_size(const MloraProjectArgs* a, int kind) {
  if (a->num_slices && a->r % 8) launch_k<T, 2, 2, kLoose>(a);
  else if (kind == kTiles128) launch_lora<T, 4, 4>(a);
  else if (kind == kTiles64x128) launch_lora<T, 2, 4>(a);
  else launch_lora<T, 2, 2>(a);
}

}  // namespace

// A tile's weights lie within 32 bits of its first, so do its rows, which with adapters may be any, and a slot's A, of up to 256 ranks.
bool tiles8_supported(const MloraProjectArgs* a) {
  static_assert(MLORA_MAX_RANK <= 1024, "a slot's A");
  return a->k <= 1 << 20 && a->x_row >= 0 && a->w_row >= 0 && a->x_row <= 1 << 22 && a->w_row <= 1 << 22 && static_cast<int64_t>(a->num_rows) * a->x_row + a->k < 1ll << 32;
}

int launch_tiles8(const MloraProjectArgs* a, int kind) {
  if (a->dtype == MLORA_DTYPE_BF16) launch_size<__bf16>(a, kind);
  else launch_size<_Float16>(a, kind);
  return check_launch("tiles8");
}

}  // namespace mlora
