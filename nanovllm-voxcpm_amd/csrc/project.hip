// The linear over 8-bit rows and weights with the adapters of many requests beside it (mlora_project), and its entry point.
//
//   y[t, n] = xs[t] ws[n] sum_k x8[t, k] w8[n, k] + bias[n] + sum_j h[t, j] B[slot of t, n, j]
//
// The base product runs on the 16x16x128 e4m3 matrix instruction, weights as its rows, so that a lane holds consecutive columns of one row of y.  The contraction of the adapters' second
// product is a list of pieces of eight ranks, those of the different slots among sixteen rows one behind the other, in which a row's h is zero outside its own slot's; it has accumulators of its own, and
// a row's pieces are added in the order of its ranks wherever its slot stands in the list: a row's result does not depend on which adapters the rows beside it have (but for one of infinities or NaN, beside which
// the row's sum is taken in another order).
//
// Few rows are bound by the weights' way to the compute units: 64 rows, k 1024, n 8192 6.0 us (8.4 MB; with 32 slots of rank 32, 21 MB more, 17), 201 rows, k 8192, n 2048 17 us (all workgroups together take 200 MB from L2 in that time, 46 bytes a ns
// each; with 48 fp16 slots of rank 64, 63 MB more, 41 us, of which the first product 12.5), one row 3.6 us, with its adapter 7.0.
#include "common.h"
#include "dma.h"
#include "launch.h"
#include "lds.h"
#include "project.h"

namespace mlora {

namespace {

// 16 NF columns of y, 16 TF rows.
//
// A stage is 128 columns of K for each of kSplit = 8 / TF wavefronts a block of sixteen rows has; stages come by direct loads, whole 128-byte lines, into a ring in LDS as deep as it holds,
// so that for K up to some thousand everything is asked for at once.  A wavefront multiplies one block of rows with all columns of its share of a stage; the shares meet in LDS at the end.
// The adapters follow as more stages: pieces of eight ranks of one of the different slots among a block's sixteen rows go to the block's wavefronts in turn, four of them a product (of one slot, or of four or two whole slots
// of one piece or two), and a stage holds each wavefront's own B and h.  (Ranks that are no multiple of eight, whose rows of B lie anywhere, are loaded by the lanes behind the last stage.)
//
// Rows in four blocks (more than 32, up to kSorted) are taken in the order of their slots where there are eight slots or more; every workgroup works the order out for itself.  The sixteen rows of a block then
// have few different slots.  (us in their own order / sorted, bf16: 256 rows, k 1024, n 1536, 48 slots of rank 64 36.9 / 27.6, 8 of rank 32 21.8 / 21.4, one slot of eight 17.3 / 21.0; 64 rows, k 2048, n 2048,
// 16 slots of rank 64 21.0 / 18.0, k 1024, n 8192, 32 of rank 32 17.1 / 16.0; 201 rows of 48 fp16 slots of rank 64, k 8192, n 2048 49.0 / 41.7.  Two blocks, 32 rows, k 1024, n 8192, 8 slots of rank 32, lost when they
// were tried: 11.8 / 12.3.)
constexpr int kRowWaves = 8, kSorted = 256;

template <int TF, int NF, int LORA> struct RowsShape {
  static constexpr int kSplit = kRowWaves / TF, kRows = 16 * (TF + NF);
  static constexpr int kPer = (kRows * 128 * kSplit + 1024 * kRowWaves - 1) / (1024 * kRowWaves);  // loads of a wavefront in a stage of the base product (as many for every one: some of nothing)
  static constexpr int kExtra = NF + 2, kMore = LORA == kStaged && kExtra > kPer ? kExtra - kPer : 0;  // in one of the adapters: B, and both parts of h
  static constexpr int kStage = (kPer + kMore) * 1024 * kRowWaves;
  static constexpr int kRing = kStage > 40 * 1024 ? 3 : kStage > 24 * 1024 ? 4 : 6;
  static constexpr int kMost = kRing * kStage, kOrder = kMost + 64, kLds = kOrder + (TF == 4 ? kSorted * 4 : 0);  // (behind the ring: the blocks' numbers of groups, the rows' order)
  static_assert(kLds <= kMostLds && 2 * kRowWaves * NF * 1024 + 64 * TF <= kMost && NF < kPer, "stages");
};

// The column of y that row `at` of a workgroup's weights is: a lane ends up with 4 NF of them side by side.
template <int NF> __device__ __forceinline__ int column_of(int at) { return 4 * NF * ((at & 15) >> 2) + 4 * (at >> 4) + (at & 3); }

// The numbers of up to kSorted rows, those of a slot side by side, rows without one last: a row's place is how many come before it, which two threads count.
__device__ __forceinline__ void sort_rows(const MloraProjectArgs& a, int32_t* keys, int32_t* order) {
  static_assert(kRowWaves * 64 == 2 * kSorted, "two threads a row");
  const int t = threadIdx.x % kSorted, half = threadIdx.x / kSorted;
  uint32_t key = 0xffffffffu;  // (the slot, then the row: no two alike)
  if (t < a.num_rows) {
    const int s = slot_of(a, t);
    key = static_cast<uint32_t>(s < 0 ? MLORA_MAX_SLOTS : s) * kSorted + t;
  }
  if (half == 0) keys[t] = static_cast<int32_t>(key);
  __syncthreads();
  int before = 0;
  if (t < a.num_rows) {
    for (int i = 16 * half; i < a.num_rows; i += 32) {
#pragma unroll
      for (int v = 0; v < 16; v += 4) {
        const i32x4 others = *reinterpret_cast<const i32x4*>(keys + i + v);
#pragma unroll
        for (int e = 0; e < 4; ++e) before += static_cast<uint32_t>(others[e]) < key;
      }
    }
  }
  if (half == 0) keys[kSorted + t] = before;
  __syncthreads();
  if (half == 1 && t < a.num_rows) order[keys[kSorted + t] + before] = t;
  __syncthreads();
}

template <typename T, int TF, int NF, int LORA> __global__ __launch_bounds__(kRowWaves * 64) void project_rows_kernel(MloraProjectArgs a) {
  using S = RowsShape<TF, NF, LORA>;
  extern __shared__ char lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int f = wave % TF, part = wave / TF;
  const int n0 = blockIdx.x * (16 * NF), t0 = blockIdx.y * (16 * TF);
  const bool sorted = TF == 4 && LORA && a.num_slots >= 8 && a.num_rows <= kSorted;
  const int32_t* const order = reinterpret_cast<const int32_t*>(lds + S::kOrder);
  if (sorted) sort_rows(a, reinterpret_cast<int32_t*>(lds), reinterpret_cast<int32_t*>(lds + S::kOrder));
  auto row_at = [&](int t) { return sorted && t < a.num_rows ? order[t] : t; };
  const int row = row_at(t0 + 16 * f + m);
  const int mine = LORA ? slot_of(a, row) : -1;  // first of all: the adapters' loads wait for it

  // what this wavefront loads of a stage: blocks of eight rows, of x or of w
  const char* from[S::kPer];
  int column[S::kPer];  // the first of K, without the stage's
#pragma unroll
  for (int i = 0; i < S::kPer; ++i) {
    const int block = wave * S::kPer + i, share = block / (S::kRows / 8), at = (block - share * (S::kRows / 8)) * 8 + (lane >> 3);
    column[i] = share * 128 + 16 * ((lane & 7) ^ ((at >> 1) & 7));
    if (at < 16 * TF) {
      const int t = row_at(t0 + at < a.num_rows ? t0 + at : a.num_rows - 1);
      from[i] = static_cast<const char*>(a.x) + static_cast<int64_t>(t) * a.x_row;
    } else {
      const int n = n0 + column_of<NF>(at - 16 * TF);
      from[i] = static_cast<const char*>(a.w) + static_cast<int64_t>(n < a.n ? n : a.n - 1) * a.w_row;
    }
  }
  const uint32_t home = lds_address(lds) + wave * (S::kPer * 1024);
  const int stages = (a.k + 128 * S::kSplit - 1) / (128 * S::kSplit);
  int put = 0, asked = 0;
  auto request = [&]() {
    const uint32_t to = __builtin_amdgcn_readfirstlane(home + put * S::kStage);
#pragma unroll
    for (int i = 0; i < S::kPer; ++i) {
      const int k = asked * (128 * S::kSplit) + column[i];
      dma16v(from[i] + (k < a.k ? k : 0), to + i * 1024);  // (behind the end of a row: its first bytes, which nobody or a zero multiplies)
    }
    put = put == S::kRing - 1 ? 0 : put + 1;
    ++asked;
  };
#pragma unroll
  for (int i = 0; i < S::kRing - 1; ++i)
    if (i < stages) request();

  // the different slots among the block's rows: lane d (and d + 16, ...) holds the d-th, `ordinal` is which one the row's is
  const int ranks = padded_ranks(a.r), pieces = ranks / 8, width = a.num_slices * ranks;
  int list = -1, ordinal = -1, count = 0;
  if constexpr (LORA) {
    unsigned long long left = __ballot(mine >= 0) & 0xffffull;
    while (left) {
      const int s = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
      const unsigned long long has = __ballot(mine == s);
      left &= ~has;
      if (mine == s) ordinal = count;
      if (m == count) list = s;
      ++count;
    }
  }
  // Groups of four pieces, a product's: slots of one piece or two share one, others have as many of their own as they need.
  const bool packed = pieces <= 2;
  const int quarters = (pieces + 3) >> 2, shift = packed ? 3 - pieces : 0;  // a slot's groups; a group has 2^shift slots
  const int groups = packed ? (count + (1 << shift) - 1) >> shift : count * quarters;
  // The wavefront that has the first of the row's groups: the others follow it in turn.
  const int leader = (packed ? ordinal >> shift : ordinal * quarters) & (S::kSplit - 1);
  auto meeting = [&](int s) {  // the first slice from s on that the columns meet
    while (s < a.num_slices && (n0 + 16 * NF <= a.slices[s].y_col || n0 >= a.slices[s].y_col + a.slices[s].n)) ++s;
    return s;
  };
  // What a lane takes of a group: piece `first` of slot d, none where `there` is not set.
  struct Place {
    int d, first;
    bool there;
  };
  auto packed_place = [&](int group) {
    const int c = 4 * group + g, d = c >> (pieces - 1);
    return Place{d, d < count ? 8 * (c - d * pieces) : 0, d < count};
  };
  auto place_in = [&](int d, int quarter) {
    const int first = 32 * quarter + 8 * g;
    return Place{d, first < ranks ? first : 0, first < ranks};
  };
  const uint16_t* const h_row = intermediate(a) + static_cast<int64_t>(row < a.num_rows ? row : a.num_rows - 1) * width;
  const int block_row = sorted ? 0 : t0 + 16 * f < a.num_rows ? t0 + 16 * f : a.num_rows - 1;  // (a block behind the last row: its loads are of that)
  const char* const h_block = reinterpret_cast<const char*>(intermediate(a) + static_cast<int64_t>(block_row) * width);
  const uint32_t h_lane = static_cast<uint32_t>((row < a.num_rows ? row - block_row : a.num_rows - 1 - block_row) * width * 2);
  // Of a slice: where its B is, how far apart two slots are in it, and the lane's rows (any for a column that is none of the slice's).
  struct Slice {
    const T* b;
    uint32_t slot_stride, in[NF];
    bool whole;
  };
  auto slice_of = [&](int s) {
    const int columns = a.slices[s].n, first = n0 - a.slices[s].y_col;
    Slice of;
    of.b = static_cast<const T*>(a.slices[s].b);
    of.slot_stride = static_cast<uint32_t>(columns) * static_cast<uint32_t>(a.r);
    of.whole = first >= 0 && first + 16 * NF <= columns;
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      const int in = first + column_of<NF>(16 * n + m);
      of.in[n] = static_cast<uint32_t>(in < 0 ? 0 : in < columns ? in : columns - 1) * static_cast<uint32_t>(a.r);
    }
    return of;
  };
  // The adapters' stages, the same number for every wavefront: of each slice, as many as the block with most groups has for a wavefront.
  int rounds = 0;
  struct Extra {
    int slice, round;
    int d, quarter;  // where a slot has groups of its own: the group's slot and which of its groups it is
  };
  auto settle_quarter = [&](Extra& e) {
    if (packed) return;
    while (e.quarter >= quarters) {
      e.quarter -= quarters;
      ++e.d;
    }
  };
  Extra load_extra = {a.num_slices, 0, 0, part};
  Slice load_slice = {};
  int extras = 0;
  if constexpr (LORA == kStaged) {
    int32_t* const most = reinterpret_cast<int32_t*>(lds + S::kMost);
    if (part == 0 && lane == 0) most[f] = groups;
    wait_lds();
    stage_barrier();
    for (int i = 0; i < TF; ++i) rounds = most[i] > rounds ? most[i] : rounds;
    rounds = __builtin_amdgcn_readfirstlane((rounds + S::kSplit - 1) / S::kSplit);
    load_extra.slice = meeting(0);
    if (rounds)
      for (int s = load_extra.slice; s < a.num_slices; s = meeting(s + 1)) extras += rounds;
    if (extras) load_slice = slice_of(load_extra.slice);
    settle_quarter(load_extra);
  }
  auto advance = [&](Extra& e, Slice& slice) {
    e.quarter += S::kSplit;
    settle_quarter(e);
    if (++e.round < rounds) return;
    e.round = 0;
    e.d = 0;
    e.quarter = part;
    settle_quarter(e);
    e.slice = meeting(e.slice + 1);
    if (e.slice < a.num_slices) slice = slice_of(e.slice);
  };
  // Where the i-th of a wavefront's loads of an adapters' stage goes: those that the base product's stages do not have lie behind theirs.
  auto place_of = [&](int i) { return i < S::kPer ? wave * (S::kPer * 1024) + i * 1024 : S::kPer * 1024 * kRowWaves + (wave * S::kMore + i - S::kPer) * 1024; };
  const int64_t h_rest = static_cast<int64_t>(a.num_rows) * width;  // from one part of h to the other
  auto request_extra = [&]() {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(lds) + put * S::kStage);
    const int group = load_extra.round * S::kSplit + part;
    if (!packed && group < groups) {
      // a slot's 32 ranks: everything but the lane's row and its eight ranks (of which the last group may have fewer) is the same for all
      const uint32_t in = 64 * load_extra.quarter + 16 * g, at = in < static_cast<uint32_t>(2 * ranks) ? in : 0;
      const char* const b = reinterpret_cast<const char*>(load_slice.b + static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(list, load_extra.d))) * load_slice.slot_stride);
      const char* const h = h_block + load_extra.slice * ranks * 2;
#pragma unroll
      for (int i = 0; i < S::kExtra; ++i) {
        if (i < NF) dma16_from(uniform(b), load_slice.in[i] * 2 + at, to + place_of(i));
        else dma16_from(uniform(i == NF ? h : h + 2 * h_rest), h_lane + at, to + place_of(i));
      }
    } else {
      const Place p = packed ? packed_place(group < groups ? group : 0) : Place{0, 0, false};
      const uint16_t* const h = h_row + load_extra.slice * ranks + p.first;
      const T* const b = load_slice.b + static_cast<uint64_t>(static_cast<uint32_t>(__shfl(list, p.there ? p.d : 0, kWave))) * load_slice.slot_stride + p.first;
#pragma unroll
      for (int i = 0; i < S::kExtra; ++i) {  // (as many as of any stage; without a group, and behind the last piece, of something that is there)
        if (i < NF && count) dma16v(reinterpret_cast<const char*>(b + load_slice.in[i]), to + place_of(i));
        else dma16v(reinterpret_cast<const char*>(i <= NF ? h : h + h_rest), to + place_of(i));
      }
    }
    put = put == S::kRing - 1 ? 0 : put + 1;
    ++asked;
    advance(load_extra, load_slice);
  };
  auto request_next = [&]() {
    if (asked < stages) request();
    else if (asked < stages + extras) request_extra();
  };
  while (asked < S::kRing - 1 && asked < stages + extras) request_next();

  f32x4 acc[NF], update[NF];  // the base product, the adapters'
#pragma unroll
  for (int n = 0; n < NF; ++n) acc[n] = update[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // Four pieces of B with the block's h.  What is not the row's, or no piece, is zero in h; columns outside the slice are in B.
  auto add_group = [&](int slice, const Place& p, bool whole, Pack8(&raw)[NF], Pack8(&h)[2]) {
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NF; ++n) {
        const int in = n0 + column_of<NF>(16 * n + m) - a.slices[slice].y_col;
        if (in < 0 || in >= a.slices[slice].n) raw[n].raw = i32x4{0, 0, 0, 0};
      }
    }
    const bool own = p.there && ordinal == p.d;
#pragma unroll
    for (int v = 0; v < 2; ++v)
      if (!own) h[v].raw = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      BPiece<T> b;
      b.from(raw[n]);
      update[n] = Mma<__bf16>::run(b.hi, h[0], update[n]);
      update[n] = Mma<__bf16>::run(b.hi, h[1], update[n]);
      if constexpr (BPiece<T>::kTwo) update[n] = Mma<__bf16>::run(b.lo, h[0], update[n]);
    }
    mfma_settle(update);
  };

  const char* const share = lds + part * (S::kRows * 128) + m * 128;
  const int piece[2] = {16 * (g ^ (m >> 1)), 16 * ((4 + g) ^ (m >> 1))};
  int now = 0;
  // Waits for a stage: no more loads may be on their way than those of the stages that were asked for behind it.
  auto wait_stage = [&](int stage) {
    const int younger = asked - 1 - stage, of_extras = asked - stages < 0 ? 0 : asked - stages < younger ? asked - stages : younger;
    wait_at_most<(S::kRing - 2) * (LORA == kStaged && S::kExtra > S::kPer ? S::kExtra : S::kPer)>(S::kPer * (younger - of_extras) + S::kExtra * of_extras);
  };
  auto next_stage = [&](int stage) {  // (is there; what came before it has been read)
    wait_lds();
    wait_stage(stage);
    stage_barrier();
    request_next();
  };
  // A stage's operands come to registers while those of the one before it are multiplied.
  auto read_stage = [&](int stage, Eight& x, Eight(&w)[NF]) {
    next_stage(stage);
    const int base = (stage * S::kSplit + part) * 128;
    const char* const at = share + now * S::kStage;
    now = now == S::kRing - 1 ? 0 : now + 1;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      x.piece[p] = load128(at + f * 2048 + piece[p]);
#pragma unroll
      for (int n = 0; n < NF; ++n) w[n].piece[p] = load128(at + (TF + n) * 2048 + piece[p]);
    }
    return base;
  };
  auto multiply = [&](int base, Eight& x, const Eight(&w)[NF]) {
    if (base + 128 > a.k) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
        if (base + 64 * p + 16 * g >= a.k) x.piece[p] = i32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int n = 0; n < NF; ++n) acc[n] = mma8(w[n], x, acc[n]);
  };
  {
    Eight x[2], w[2][NF];
    int base = read_stage(0, x[0], w[0]), next = 0;
    for (int stage = 1; stage < stages; stage += 2) {
      next = read_stage(stage, x[1], w[1]);
      multiply(base, x[0], w[0]);
      if (stage + 1 >= stages) {
        x[0] = x[1];
#pragma unroll
        for (int n = 0; n < NF; ++n) w[0][n] = w[1][n];
        base = next;
        break;
      }
      base = read_stage(stage + 1, x[0], w[0]);
      multiply(next, x[1], w[1]);
    }
    multiply(base, x[0], w[0]);
    mfma_settle(acc);
  }
#pragma unroll
  for (int n = 0; n < NF; ++n) {
    const int c = n0 + 4 * NF * g + 4 * n;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] *= a.w_scales[c + i < a.n ? c + i : a.n - 1];
  }
  if (LORA == kStaged && extras) {
    Extra e = {meeting(0), 0, 0, part};
    settle_quarter(e);
    Slice slice = slice_of(e.slice);
    for (int stage = stages; stage < stages + extras; ++stage) {
      // (a wavefront reads what it has loaded itself: only the last stage of the base product has to be everybody's)
      wait_lds();
      wait_stage(stage);
      if (stage == stages) stage_barrier();
      request_next();
      const int group = e.round * S::kSplit + part;
      const char* const at = lds + now * S::kStage + lane * 16;
      now = now == S::kRing - 1 ? 0 : now + 1;
      if (group < groups) {
        Pack8 raw[NF], h[2];
#pragma unroll
        for (int n = 0; n < NF; ++n) raw[n].raw = load128(at + place_of(n));
#pragma unroll
        for (int v = 0; v < 2; ++v) h[v].raw = load128(at + place_of(NF + v));
        add_group(e.slice, packed ? packed_place(group) : place_in(e.d, e.quarter), slice.whole, raw, h);
      }
      advance(e, slice);
    }
  }
  if constexpr (LORA == kLoose) {
    for (int s = meeting(0); s < a.num_slices; s = meeting(s + 1)) {
      const Slice slice = slice_of(s);
      Extra e = {s, 0, 0, part};
      settle_quarter(e);
      for (int group = part; group < groups; group += S::kSplit) {
        const Place p = packed ? packed_place(group) : place_in(e.d, e.quarter);
        e.quarter += S::kSplit;
        settle_quarter(e);
        const T* const b_slot = slice.b + static_cast<uint64_t>(static_cast<uint32_t>(__shfl(list, p.there ? p.d : 0, kWave))) * slice.slot_stride;
        Pack8 raw[NF], h[2];
#pragma unroll
        for (int n = 0; n < NF; ++n) {
          T* const to = reinterpret_cast<T*>(&raw[n]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            to[i] = b_slot[slice.in[n] + (p.first + i < a.r ? p.first + i : 0)];
            if (p.first + i >= a.r) to[i] = static_cast<T>(0.0f);
          }
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) h[v].raw = load128(h_row + v * h_rest + s * ranks + p.first);
        add_group(s, p, slice.whole, raw, h);
      }
    }
  }
  // An infinity or a NaN in B goes through a matrix product to the rows of other slots (0 times it is NaN): where one came out the row's own adapter is added again, one number at a time.
  unsigned beyond = 0;
#pragma unroll
  for (int n = 0; n < NF; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) beyond |= (__float_as_uint(update[n][i]) & 0x7f800000u) == 0x7f800000u ? 1u << n : 0;
  if (beyond) {
#pragma unroll
    for (int n = 0; n < NF; ++n)
      if (beyond >> n & 1) update[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int ahead = (part - leader) & (S::kSplit - 1);  // which of the row's groups the wavefront has first
    if (ordinal >= 0)
      for (int s = meeting(0); s < a.num_slices; s = meeting(s + 1))
        for (int quarter = ahead; quarter < quarters; quarter += S::kSplit) {
          const T* const b = static_cast<const T*>(a.slices[s].b) + static_cast<int64_t>(mine) * a.slices[s].n * a.r;
          const uint16_t* const hi = h_row + s * ranks;
#pragma unroll
          for (int n = 0; n < NF; ++n)
            if (beyond >> n & 1)
              add_slowly(b, a.slices[s].n, n0 + 4 * NF * g + 4 * n - a.slices[s].y_col, a.r, 32 * quarter, 32, hi, hi + h_rest, update[n]);
        }
  }
  // the shares meet
  wait_lds();
  wait_loads<0>();
  __syncthreads();
  constexpr int kUpdates = kRowWaves * NF * 64;
  f32x4* const parts = reinterpret_cast<f32x4*>(lds);
  int32_t* const leaders = reinterpret_cast<int32_t*>(lds + 2 * kUpdates * 16);
#pragma unroll
  for (int n = 0; n < NF; ++n) parts[(wave * NF + n) * 64 + lane] = acc[n];
  if constexpr (LORA) {
#pragma unroll
    for (int n = 0; n < NF; ++n) parts[kUpdates + (wave * NF + n) * 64 + lane] = update[n];
    if (part == 0 && g == 0) leaders[16 * f + m] = leader;
  }
  __syncthreads();
  for (int block = wave; block < TF * NF; block += kRowWaves) {
    const int of = block / NF, c = n0 + 4 * NF * g + 4 * (block % NF);
    if (t0 + 16 * of + m >= a.num_rows || c >= a.n) continue;
    const int t = row_at(t0 + 16 * of + m);
    f32x4 sum = parts[(of * NF + block % NF) * 64 + lane];
#pragma unroll
    for (int v = 1; v < S::kSplit; ++v) sum += parts[((v * TF + of) * NF + block % NF) * 64 + lane];
    if constexpr (LORA) {
      const int first = leaders[16 * of + m];
      f32x4 added = parts[kUpdates + ((first * TF + of) * NF + block % NF) * 64 + lane];
      for (int v = 1; v < S::kSplit && v < quarters; ++v) added += parts[kUpdates + ((((first + v) & (S::kSplit - 1)) * TF + of) * NF + block % NF) * 64 + lane];
      sum += added;
    }
    const float scale = a.x_scales[t];
    T out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = from_f32<T>(__builtin_fmaf(sum[i], scale, a.bias ? to_f32(static_cast<const T*>(a.bias)[c + i < a.n ? c + i : a.n - 1]) : 0.0f));
    T* const y = static_cast<T*>(a.y) + static_cast<int64_t>(t) * a.y_row + c;
    if (c + 4 <= a.n && ((reinterpret_cast<uintptr_t>(a.y) | static_cast<uintptr_t>(a.y_row * 2)) & 7) == 0) {
      __builtin_memcpy(__builtin_assume_aligned(y, 8), out, 8);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < a.n) y[i] = out[i];
    }
  }
}

// Very few rows with their adapters in one launch: sixteen columns a workgroup, which works out the rows' whole h for itself.
//
// A second launch and the trip of h through memory cost more than every workgroup's reading of the rows' A, from L2, as long as that is little (few_rows below).  The wavefronts share K, 128 columns each in turn, of the base product and of
// h; h is added up in LDS and rounded as in the other kernels, and the first wavefront multiplies it with B, in one product: there are four pieces of eight ranks at most.
constexpr int kFewGroups = 2;  // of sixteen ranks of a slot, all rows together

template <typename T> __global__ __launch_bounds__(kRowWaves * 64) void project_few_kernel(MloraProjectArgs a) {
  __shared__ f32x4 parts[kFewGroups][kRowWaves][64];
  __shared__ __align__(16) uint16_t h_of[2][16][16 * kFewGroups];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, mine = slot_of(a, m);
  // the different slots among the rows: lane d holds the d-th, `ordinal` is which one the row's is
  int list = 0, ordinal = -1, count = 0;
  unsigned long long left = __ballot(mine >= 0) & 0xffffull;
  while (left) {
    const int s = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const unsigned long long has = __ballot(mine == s);
    left &= ~has;
    if (mine == s) ordinal = count;
    if (m == count) list = s;
    ++count;
  }
  const int ranks = padded_ranks(a.r), pieces = ranks / 8, of_slot = (ranks + 15) / 16, groups = count * of_slot, total = count * pieces;
  const char* const x = static_cast<const char*>(a.x) + static_cast<int64_t>(m < a.num_rows ? m : a.num_rows - 1) * a.x_row;
  const char* const w = static_cast<const char*>(a.w) + static_cast<int64_t>(n0 + m < a.n ? n0 + m : a.n - 1) * a.w_row;
  f32x4 acc[1] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
  auto meets = [&](int s) { return n0 < a.slices[s].y_col + a.slices[s].n && n0 + 16 > a.slices[s].y_col; };
  // The lane's piece of the contraction: eight ranks of the d-th slot, from `first` on.
  const int d = g / pieces, first = 8 * (g - d * pieces), slot = __shfl(list, g < total ? d : 0, kWave);
  // of a lane's piece behind the last column the row's first one is read, and nothing kept
  auto load_x = [&](int k, Eight& to) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int at = k + 64 * p + 16 * g;
      to.piece[p] = load128(x + (at < a.k ? at : 0));
      if (at >= a.k) to.piece[p] = i32x4{0, 0, 0, 0};
    }
  };
  for (int k = wave * 128; k < a.k; k += kRowWaves * 128) {
    Eight xs, ws;
    load_x(k, xs);
#pragma unroll
    for (int p = 0; p < 2; ++p) ws.piece[p] = load128(w + (k + 64 * p + 16 * g < a.k ? k + 64 * p + 16 * g : 0));
    acc[0] = mma8(ws, xs, acc[0]);
  }
  mfma_settle(acc);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[0][i] *= a.w_scales[n0 + 4 * g + i < a.n ? n0 + 4 * g + i : a.n - 1];
  for (int s = 0; s < a.num_slices; ++s) {
    if (!meets(s)) continue;
    Pack8 b;  // (on its way while h comes about; zero where there is no piece, or the column is none of the slice's)
    b.raw = i32x4{0, 0, 0, 0};
    const int in = n0 + m - a.slices[s].y_col;
    if (wave == 0 && g < total && in >= 0 && in < a.slices[s].n) b.raw = load128(static_cast<const T*>(a.slices[s].b) + (static_cast<int64_t>(slot) * a.slices[s].n + in) * a.r + first);
    const T* rows[kFewGroups];
#pragma unroll
    for (int v = 0; v < kFewGroups; ++v) {
      const int of = v < groups ? v : 0, its = of / of_slot, j = (of - its * of_slot) * 16 + m;
      rows[v] = static_cast<const T*>(a.slices[s].a) + (static_cast<int64_t>(__builtin_amdgcn_readlane(list, its)) * a.r + (j < a.r ? j : a.r - 1)) * a.k;
    }
    f32x4 h[kFewGroups];
#pragma unroll
    for (int v = 0; v < kFewGroups; ++v) h[v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = wave * 128; k < a.k && groups; k += kRowWaves * 128) {
      Eight xs;
      load_x(k, xs);
      Pack8 as[kFewGroups][2][2];
#pragma unroll
      for (int v = 0; v < kFewGroups; ++v)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int at = k + 64 * p + 16 * g < a.k ? k + 64 * p + 16 * g : 0;
          as[v][p][0].raw = load128(rows[v] + at);
          as[v][p][1].raw = load128(rows[v] + at + 8);
        }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        Pack8 wide[2];
        widen<T>(xs.piece[p], wide);
        const bool there = k + 64 * p + 16 * g < a.k;
#pragma unroll
        for (int v = 0; v < kFewGroups; ++v)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (!there) as[v][p][e].raw = i32x4{0, 0, 0, 0};
            h[v] = Mma<T>::run(as[v][p][e], wide[e], h[v]);
          }
      }
    }
    mfma_settle(h);
#pragma unroll
    for (int v = 0; v < kFewGroups; ++v) parts[v][wave][lane] = h[v];
    __syncthreads();
    if (wave < groups) {  // a wavefront adds up one group's
      f32x4 sum = parts[wave][0][lane];
#pragma unroll
      for (int v = 1; v < kRowWaves; ++v) sum += parts[wave][v][lane];
      const int its = wave / of_slot, j = (wave - its * of_slot) * 16 + 4 * g;
      if (ordinal == its) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          __bf16 hi, lo;
          split(j + i < a.r ? sum[i] : 0.0f, &hi, &lo);
          h_of[0][m][j + i] = __builtin_bit_cast(uint16_t, hi);
          h_of[1][m][j + i] = __builtin_bit_cast(uint16_t, lo);
        }
      }
    }
    __syncthreads();
    if (wave == 0 && total) {
      const f32x4 before = acc[0];
      const bool own = g < total && ordinal == d;
      BPiece<T> of;
      of.from(b);
      Pack8 h;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        h.raw = own ? load128(&h_of[v][m][first]) : i32x4{0, 0, 0, 0};
        acc[0] = Mma<__bf16>::run(of.hi, h, acc[0]);
        if constexpr (BPiece<T>::kTwo)
          if (v == 0) acc[0] = Mma<__bf16>::run(of.lo, h, acc[0]);
      }
      mfma_settle(acc);
      // (infinities and NaN in B: see the kernel above)
      bool beyond = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) beyond |= (__float_as_uint(acc[0][i]) & 0x7f800000u) == 0x7f800000u;
      if (beyond) {
        acc[0] = before;
        if (ordinal >= 0)
          add_slowly(static_cast<const T*>(a.slices[s].b) + static_cast<int64_t>(mine) * a.slices[s].n * a.r, a.slices[s].n, n0 + 4 * g - a.slices[s].y_col, a.r, 0, a.r, h_of[0][m],
                     h_of[1][m], acc[0]);
      }
    }
    __syncthreads();  // (the next slice has another h)
  }
  parts[0][wave][lane] = acc[0];
  __syncthreads();
  if (wave || m >= a.num_rows) return;
  f32x4 sum = parts[0][0][lane];
#pragma unroll
  for (int v = 1; v < kRowWaves; ++v) sum += parts[0][v][lane];
  const float scale = a.x_scales[m];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = n0 + 4 * g + i;
    if (c < a.n) static_cast<T*>(a.y)[static_cast<int64_t>(m) * a.y_row + c] = from_f32<T>(__builtin_fmaf(sum[i], scale, a.bias ? to_f32(static_cast<const T*>(a.bias)[c]) : 0.0f));
  }
}

// The rows' A of at most two times sixteen ranks, a K of two turns, and few enough workgroups that they do not wait for each other in L2: as in one launch / in two, us, graph replay, 1 row, rank 32: k 1024,
// n 1536 7.0 / 9.4, n 8192 9.4 / 10.4; k 2048, n 2048 9.4 / 11.0, n 8192 14.2 / 12.6; k 4096, n 1024 13.9 / 13.5; of rank 64 (four times sixteen), when it was tried, k 1024, n 1536 8.8 / 8.9, n 8192 13.0 / 9.8.
bool few_rows(const MloraProjectArgs* a) {
  return a->num_slices && a->r % 8 == 0 && a->num_rows <= kFewGroups && a->num_rows * ((a->r + 15) / 16) <= kFewGroups && a->k <= 2048 && static_cast<int64_t>(a->n) * a->k <= 1 << 23;
}

template <typename T, int TF, int NF, int LORA> void launch_ranks(const MloraProjectArgs* a) {
  constexpr int bytes = RowsShape<TF, NF, LORA>::kLds;
  allow_lds<project_rows_kernel<T, TF, NF, LORA>>(bytes);
  const dim3 grid(static_cast<unsigned>((a->n + 16 * NF - 1) / (16 * NF)), static_cast<unsigned>((a->num_rows + 16 * TF - 1) / (16 * TF)));
  project_rows_kernel<T, TF, NF, LORA><<<grid, kRowWaves * 64, bytes, static_cast<hipStream_t>(a->stream)>>>(*a);
}
template <typename T, int TF, int NF> void launch(const MloraProjectArgs* a) {
  if (!a->num_slices) launch_ranks<T, TF, NF, kNone>(a);
  else if (a->r % 8) launch_ranks<T, TF, NF, kLoose>(a);
  else launch_ranks<T, TF, NF, kStaged>(a);
}
template <typename T, int TF> void launch_columns(const MloraProjectArgs* a) {
  // 32 columns a workgroup where that still gives every compute unit one
  const int64_t wide = static_cast<int64_t>((a->n + 31) / 32) * ((a->num_rows + 16 * TF - 1) / (16 * TF));
  if (wide >= 256) launch<T, TF, 2>(a);
  else launch<T, TF, 1>(a);
}
template <typename T> void launch_few(const MloraProjectArgs* a) {
  project_few_kernel<T><<<static_cast<unsigned>((a->n + 15) / 16), kRowWaves * 64, 0, static_cast<hipStream_t>(a->stream)>>>(*a);
}
template <typename T> void launch_rows(const MloraProjectArgs* a) {
  if (a->num_rows <= 16) launch_columns<T, 1>(a);
  else if (a->num_rows <= 32) launch_columns<T, 2>(a);
  else launch_columns<T, 4>(a);
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

size_t workspace_bytes(const MloraProjectArgs* a) {
  return static_cast<size_t>(order_bytes(a->num_rows, a->num_slots)) + static_cast<size_t>(a->num_rows) * a->num_slices * padded_ranks(a->r) * 4;
}

int check_project(const MloraProjectArgs* a) {
  const char* const what = "mlora_project";
  if (!a) { set_error("%s: NULL args", what); return MLORA_E_INVALID; }
  if (a->num_rows < 0 || a->k < 0 || a->n < 0 || a->num_slices < 0 || a->r < 0 || a->num_slots < 0) { set_error("%s: negative size", what); return MLORA_E_INVALID; }
  if (a->dtype != MLORA_DTYPE_F16 && a->dtype != MLORA_DTYPE_BF16) { set_error("%s: dtype %d is neither fp16 nor bf16", what, a->dtype); return MLORA_E_UNSUPPORTED; }
  if (a->k % 16) { set_error("%s: k = %d is not a multiple of 16", what, a->k); return MLORA_E_UNSUPPORTED; }
  if (a->num_slices > MLORA_MAX_SLICES || a->num_slots > MLORA_MAX_SLOTS || a->r > MLORA_MAX_RANK) {
    set_error("%s: %d slices, %d slots, rank %d: at most %d, %d, %d", what, a->num_slices, a->num_slots, a->r, MLORA_MAX_SLICES, MLORA_MAX_SLOTS, MLORA_MAX_RANK);
    return MLORA_E_TOO_LARGE;
  }
  if (a->num_rows == 0 || a->n == 0) return kNothingToDo;
  if (a->k == 0) { set_error("%s: rows without elements", what); return MLORA_E_INVALID; }
  if (a->k > 1 << 22 || a->n > 1 << 22 || a->num_rows > 1 << 20) { set_error("%s: %d rows, k = %d, n = %d: at most 2^20, 2^22, 2^22", what, a->num_rows, a->k, a->n); return MLORA_E_TOO_LARGE; }
  if (!a->x || !a->x_scales || !a->w || !a->w_scales || !a->y) { set_error("%s: NULL pointer", what); return MLORA_E_INVALID; }
  if (!on16(a->x) || !on16(a->w) || a->x_row % 16 || a->w_row % 16) { set_error("%s: rows of x and w must start on 16 bytes", what); return MLORA_E_INVALID; }
  if (a->num_slices == 0) return 0;
  if (a->num_slots == 0 || a->r == 0) { set_error("%s: adapters without slots or ranks", what); return MLORA_E_INVALID; }
  if (!a->token_to_slot) { set_error("%s: token_to_slot is NULL", what); return MLORA_E_INVALID; }
  int end = 0;
  for (int s = 0; s < a->num_slices; ++s) {
    const MloraSlice& slice = a->slices[s];
    if (slice.n < 1 || slice.y_col < end || slice.y_col > a->n - slice.n) {
      set_error("%s: slice %d of %d columns from %d on does not lie behind the one before it, inside %d", what, s, slice.n, slice.y_col, a->n);
      return MLORA_E_INVALID;
    }
    end = slice.y_col + slice.n;
    if (!slice.a || !slice.b || !on16(slice.a) || !on16(slice.b)) { set_error("%s: a and b of slice %d must start on 16 bytes", what, s); return MLORA_E_INVALID; }
  }
  if (!a->workspace || !on16(a->workspace) || a->workspace_bytes < static_cast<int64_t>(workspace_bytes(a))) {
    set_error("%s: workspace of %lld bytes, %zu are needed, on 16 bytes", what, static_cast<long long>(a->workspace_bytes), workspace_bytes(a));
    return MLORA_E_INVALID;
  }
  return 0;
}

}  // namespace

// Rows by themselves up to 64, and up to 256 while their workgroups are no more than the compute units: what they share out along K a tile has to go through alone, and tiles want the rows in
// the order of their slots first; beyond, a second round of them costs a base product as much as the first.  (us, graph replay, bf16, 8 slots of rank 32, random; in brackets without adapters:
// 128 rows, k 4096, n 4096, 256 workgroups: 24.3 [10.6], by tiles 38.1 [12.5]; 192 rows: 36.9 [18.9], 37.4 [13.1]; 96 rows, k 1024, n 8192, 512 workgroups: 21.7 [9.6], 24.5 [6.1].  Of short K the rule gives up
// without adapters about what it gains with them: 256 rows, k 1024, n 1536 21.2 [8.3], 23.2 [5.8]; 192 rows, k 2048, n 2048 23.9 [10.6], 27.7 [7.9].)
// Of the tiles the smallest that are all at work at once, 64 x 64 three a compute unit, 64 x 128 three or, with adapters, two, else 128 x 128, which loads least.  (k 4096, n 4096: 768 rows
// 20.5 / 22.9 / 25.7 without adapters, 45.8 / 46.5 / 52.0 with; 1024 rows 25.3 / 23.0 / 25.6, 60.8 / 46.6 / 50.7; 2048 rows 48.7 / 45.1 / 34.8, 99.1 / 72.4 / 61.4.)
// Which of the tiles changes nothing in the result: all go through K in the same steps.
int project_kind(const MloraProjectArgs* a) {
  auto tiles = [&](int rows, int columns) { return static_cast<int64_t>((a->num_rows + rows - 1) / rows) * ((a->n + columns - 1) / columns); };
  if (a->num_rows <= 64 || (a->num_rows <= 256 && tiles(64, 32) <= 256) || !tiles8_supported(a)) return kRows;
  if (tiles(64, 64) <= 3 * 256) return kTiles64;
  return tiles(64, 128) <= (a->num_slices ? 2 : 3) * 256 ? kTiles64x128 : kTiles128;
}

int launch_project_rows(const MloraProjectArgs* a) {
  if (a->dtype == MLORA_DTYPE_BF16) launch_rows<__bf16>(a);
  else launch_rows<_Float16>(a);
  return check_launch("project");
}

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_project(const MloraProjectArgs* a) {
  const int rc = check_project(a);
  if (rc) return rc == kNothingToDo ? 0 : rc;
  if (few_rows(a)) {
    if (a->dtype == MLORA_DTYPE_BF16) launch_few<__bf16>(a);
    else launch_few<_Float16>(a);
    return check_launch("project");
  }
  const int kind = project_kind(a);
  if (a->num_slices)
    if (const int failed = launch_shrink8(a, kind != kRows)) return failed;
  return kind == kRows ? launch_project_rows(a) : launch_tiles8(a, kind);
}

extern "C" size_t mlora_project_workspace_bytes(const MloraProjectArgs* a) {
  return a && a->num_rows > 0 && a->n > 0 && a->num_slices > 0 && a->num_slices <= MLORA_MAX_SLICES && a->r > 0 && a->r <= MLORA_MAX_RANK ? workspace_bytes(a) : 0;
}
