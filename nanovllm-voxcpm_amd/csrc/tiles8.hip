// The 8-bit linear over tiles of rows and columns, for many rows (see project.hip for the formula, project.h for the operands).
//
// Four wavefronts have a tile of y, each a quarter.  128 columns of K of the tile's rows and weights come by direct loads into one of two buffers in LDS, two steps
// ahead of the products and on into the workgroup's next tile, so that the loads of a tile's beginning run under the end of the one before it.  A load takes
// whole 128-byte lines of eight rows: with halves of lines of sixteen rows, which want no exchange in LDS, every line was fetched twice (8192 x 8192 x 8192: 655 us; this way 463).
#include "common.h"
#include "dma.h"
#include "launch.h"
#include "lds.h"
#include "project.h"

namespace mlora {

namespace {

constexpr int kXcds = 8;

struct Tile {
  int t, n;
};
// Which tile comes `id`-th.  Workgroups go to the eight XCDs in turn; each XCD gets a run of tiles, in strips of eight row tiles, columns by columns, so that what
// works on an XCD at one time shares rows and columns in its L2.
__device__ __forceinline__ Tile tile_of(int id, int rows, int columns) {
  const int total = rows * columns, share = total / kXcds, more = total % kXcds, xcd = id % kXcds;
  const int at = xcd * share + (xcd < more ? xcd : more) + id / kXcds;
  constexpr int kStrip = 8;
  const int strip = at / (kStrip * columns), in = at - strip * (kStrip * columns);
  const int high = rows - strip * kStrip < kStrip ? rows - strip * kStrip : kStrip;
  return Tile{strip * kStrip + in % high, in / high};
}

template <typename T, int TT, int NN, bool TAIL, bool LORA> __global__ __launch_bounds__(256, LORA || TT * NN > 8 ? 2 : 3) void tiles8_kernel(MloraProjectArgs a) {
  constexpr int BT = 32 * TT, BN = 32 * NN, kStage = (BT + BN) * 128;
  extern __shared__ char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wt = wave >> 1, wn = wave & 1;
  const int rows = (a.num_rows + BT - 1) / BT, columns = (a.n + BN - 1) / BN, total = rows * columns;
  const uint32_t home = lds_address(lds);

  // the loads run two steps ahead of the products, over the tiles of this workgroup one behind the other
  int load_tile = blockIdx.x, load_k = 0, buffer = 0;
  const char *x_base = nullptr, *w_base = nullptr;
  // rows in the order of their slots
  const int32_t* const order = static_cast<const int32_t*>(a.workspace);
  int coming[TT];  // the rows that this lane loads of the tile after the next
  auto look_up = [&](int id) {
    if (id >= total) return;
    const int t0 = tile_of(id, rows, columns).t * BT;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int at = t0 + (wave * TT + i) * 8 + (lane >> 3);
      coming[i] = order[at < a.num_rows ? at : a.num_rows - 1];
    }
  };
  uint32_t x_off[TT], w_off[NN];  // eight rows a load, whole lines of 128 bytes; a row's 16-byte pieces lie exchanged in LDS
  auto aim = [&]() {
    const Tile tile = tile_of(load_tile, rows, columns);
    const int t0 = tile.t * BT, n0 = tile.n * BN;
    x_base = static_cast<const char*>(a.x) + (LORA ? 0 : static_cast<int64_t>(t0) * a.x_row);
    w_base = static_cast<const char*>(a.w) + static_cast<int64_t>(n0) * a.w_row;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int row = (wave * TT + i) * 8 + (lane >> 3), most = a.num_rows - t0 - 1;
      x_off[i] = static_cast<uint32_t>((LORA ? coming[i] : row < most ? row : most) * a.x_row);
    }
    if constexpr (LORA) look_up(load_tile + gridDim.x);
#pragma unroll
    for (int i = 0; i < NN; ++i) {
      const int at = (wave * NN + i) * 8 + (lane >> 3), block = at >> 4, f = block % NN, r = at & 15, most = a.n - n0 - 1;
      const int row = block / NN * (16 * NN) + 32 * (f >> 1) + 8 * (r >> 2) + 4 * (f & 1) + (r & 3);
      w_off[i] = static_cast<uint32_t>((row < most ? row : most) * a.w_row);
    }
  };
  auto request = [&]() {
    if (load_tile >= total) return;
    if (load_k == 0) aim();  // (everything that was asked for is there: the rows to load as well)
    const uint32_t to = home + buffer * kStage;
    // piece c of row r lies at c ^ (r / 2 % 8): sixteen rows' same piece, which a product reads at once, in all banks
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {  // (rows 8 .. 15 of a block of sixteen)
      const int k = load_k + 16 * ((lane & 7) ^ (((lane >> 4) & 3) + 4 * odd));
      const uint32_t at = !TAIL || k < a.k ? k : 0;  // (behind the end of a row: its first bytes, which are multiplied by zero)
#pragma unroll
      for (int i = odd; i < TT; i += 2) dma16(x_base, x_off[i] + at, to + (wave * TT + i) * 1024);
#pragma unroll
      for (int i = odd; i < NN; i += 2) dma16(w_base, w_off[i] + at, to + (4 * TT + wave * NN + i) * 1024);
    }
    buffer ^= 1;
    load_k += 128;
    if (load_k >= a.k) {
      load_k = 0;
      load_tile += gridDim.x;
    }
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
  // One step: its blocks of w and the first two of x are in registers; leaves the next step's there.
  auto step = [&](Eight(&w)[NN], Eight(&x01)[2], Eight(&next_w)[NN], Eight(&next_x)[2]) {
    const char* const xs = x_home + now * kStage;
    Eight x[TT];
    x[0] = x01[0];
    x[1] = x01[1];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      if (t + 2 < TT) block_of(xs, t + 2, x[t + 2]);
      if (t == TT - 2) {
        // everything of this step has been read: its buffer takes the step after the next, which is there
        wait_lds();
        wait_loads<0>();
        stage_barrier();
        request();
        const int other = (now ^ 1) * kStage;
#pragma unroll
        for (int n = 0; n < NN; ++n) block_of(w_home + other, n, next_w[n]);
#pragma unroll
        for (int i = 0; i < 2; ++i) block_of(x_home + other, i, next_x[i]);
      }
      if constexpr (TAIL) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (k + 64 * p + 16 * g >= a.k) x[t].piece[p] = i32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int n = 0; n < NN; ++n) acc[t][n] = mma8(w[n], x[t], acc[t][n]);
    }
    // (the last results may be read behind a branch that leaves the loop: the wait for a matrix instruction, which the next one would have to keep as well)
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    k += 128;
    now ^= 1;
  };

  if constexpr (LORA) look_up(load_tile);
  request();
  wait_loads<0>();
  stage_barrier();
  request();
  Eight w[2][NN], x01[2][2];
  auto begin = [&]() {
#pragma unroll
    for (int n = 0; n < NN; ++n) block_of(w_home + now * kStage, n, w[0][n]);
#pragma unroll
    for (int i = 0; i < 2; ++i) block_of(x_home + now * kStage, i, x01[0][i]);
  };
  begin();
  for (int id = blockIdx.x; id < total; id += gridDim.x) {
    if (LORA && id != blockIdx.x) begin();  // (again: the adapters want the registers)
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int n = 0; n < NN; ++n) acc[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (k = 0; k < a.k;) {
      step(w[0], x01[0], w[1], x01[1]);
      if (k < a.k) {
        step(w[1], x01[1], w[0], x01[0]);
      } else {
#pragma unroll
        for (int n = 0; n < NN; ++n) w[0][n] = w[1][n];
#pragma unroll
        for (int i = 0; i < 2; ++i) x01[0][i] = x01[1][i];
      }
    }

    const Tile tile = tile_of(id, rows, columns);
    const int t0 = tile.t * BT + wt * (16 * TT), n0 = tile.n * BN + wn * (16 * NN) + 8 * g;  // the lane's columns: n0 + 32 c + 0 .. 7
    const bool whole = (tile.n + 1) * BN <= a.n && ((reinterpret_cast<uintptr_t>(a.y) | static_cast<uintptr_t>(a.y_row * 2)) & 15) == 0;
    int mine[TT];
    if constexpr (LORA) {
      const int32_t* const slots = order + a.num_rows;
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const int at = t0 + 16 * t + m;
        mine[t] = slots[at < a.num_rows ? at : a.num_rows - 1];
        if (at >= a.num_rows) mine[t] = -1;
      }
    }
    float scales[NN / 2][8];
#pragma unroll
    for (int c = 0; c < NN / 2; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) scales[c][i] = a.w_scales[n0 + 32 * c + i < a.n ? n0 + 32 * c + i : a.n - 1];
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int n = 0; n < NN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][n][i] *= scales[n / 2][n % 2 * 4 + i];

    if constexpr (LORA) {  // every different slot among the wavefront's rows
      const int ranks = padded_ranks(a.r), width = a.num_slices * ranks;
      const uint16_t* const hi = intermediate(a);
      const uint16_t* const lo = hi + static_cast<int64_t>(a.num_rows) * width;
      const bool words = a.r % 8 == 0;
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
              if (words) {
                raw[n].raw = load128(from);
              } else {
                T* e = reinterpret_cast<T*>(&raw[n]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  e[i] = from[there && rank + i < a.r ? i : 0];
                  if (rank + i >= a.r) e[i] = static_cast<T>(0.0f);
                }
              }
              if (!there) raw[n].raw = i32x4{0, 0, 0, 0};
            }
            BPiece<T> b[NN];
#pragma unroll
            for (int n = 0; n < NN; ++n) b[n].from(raw[n]);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
              if (!has[t]) continue;
              // (a lane's results are of one row, and come from that row's h alone: rows of other slots keep what they have, whatever is in this one's B)
              const bool own = mine[t] == slot;
#pragma unroll
              for (int n = 0; n < NN; ++n) {
                f32x4 next = Mma<__bf16>::run(b[n].hi, h[t][0], acc[t][n]);
                next = Mma<__bf16>::run(b[n].hi, h[t][1], next);
                if constexpr (BPiece<T>::kTwo) next = Mma<__bf16>::run(b[n].lo, h[t][0], next);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][n][i] = own ? next[i] : acc[t][n][i];
              }
            }
          }
        }
      }
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
      const int row = LORA ? order[at] : at;
      const float scale = a.x_scales[row];
      T* const y = static_cast<T*>(a.y) + static_cast<int64_t>(row) * a.y_row + n0;
#pragma unroll
      for (int c = 0; c < NN / 2; ++c) {
        T out[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = from_f32<T>(__builtin_fmaf(acc[t][2 * c + i / 4][i % 4], scale, bias[c][i]));
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
  }
}

template <typename T, int TT, int NN, bool TAIL, bool LORA> void launch(const MloraProjectArgs* a) {
  constexpr auto kernel = tiles8_kernel<T, TT, NN, TAIL, LORA>;
  constexpr int bytes = 2 * (32 * TT + 32 * NN) * 128;
  allow_lds<kernel>(bytes);
  const int64_t tiles = static_cast<int64_t>((a->num_rows + 32 * TT - 1) / (32 * TT)) * ((a->n + 32 * NN - 1) / (32 * NN));
  const int64_t most = 256 * (TT * NN > 8 ? 2 : TT * NN > 4 ? 3 : 4);
  kernel<<<static_cast<unsigned>(tiles < most ? tiles : most), 256, bytes, static_cast<hipStream_t>(a->stream)>>>(*a);
}
template <typename T, int TT, int NN> void launch_k(const MloraProjectArgs* a) {
  if (a->num_slices) {
    if (a->k % 128) launch<T, TT, NN, true, true>(a);
    else launch<T, TT, NN, false, true>(a);
  } else {
    if (a->k % 128) launch<T, TT, NN, true, false>(a);
    else launch<T, TT, NN, false, false>(a);
  }
}
template <typename T> void launch_size(const MloraProjectArgs* a, int kind) {
  if (kind == kTiles128) launch_k<T, 4, 4>(a);
  else if (kind == kTiles64x128) launch_k<T, 2, 4>(a);
  else launch_k<T, 2, 2>(a);
}

}  // namespace

// A tile's weights lie within 32 bits of its first, and so do its rows, which with adapters may be any.
bool tiles8_supported(const MloraProjectArgs* a) {
  return a->x_row >= 0 && a->w_row >= 0 && a->x_row <= 1 << 22 && a->w_row <= 1 << 22 && static_cast<int64_t>(a->num_rows) * a->x_row + a->k < 1ll << 32;
}

int launch_tiles8(const MloraProjectArgs* a, int kind) {
  if (a->dtype == MLORA_DTYPE_BF16) launch_size<__bf16>(a, kind);
  else launch_size<_Float16>(a, kind);
  return check_launch("tiles8");
}

}  // namespace mlora
