// Attention of packed prompts over packed or paged keys, head sizes 64 and 128 (mlora_prompt_attention).
//
// One workgroup per 128 rows of queries that share a key-value head: four wavefronts of 32 rows each, of one head or of several.  Tiles of 64 keys and their values are
// staged in LDS by direct loads, two stages deep: one barrier a tile, behind which the next tile is asked for.  The scores come out of the first product with the
// keys along the registers and the query rows along the lanes (K Q^T, 32 x 32 tiles), which is how the second one (V^T P^T) wants its
// weights: they never leave the registers, a row's maximum and sum are a lane's own but for one exchange between the halves of the
// wave, and V^T is read through the transposing LDS read.  The running maximum moves only when a tile's exceeds it by more than 2^8
// (any base serves a softmax as long as its weights stay finite), so the outputs are hardly ever rescaled.
//
// Bound by the matrix cores and what stands between their two products.  At head size 64 a tile of 64 keys costs a wavefront 512 cycles of matrix core, 256 of
// exponentials (32 of 8 cycles) and 250 of the other vector instructions (two cycles each where wavefronts share a SIMD); three wavefronts a SIMD overlap them, and the
// matrix cores are busy for 45 % of the cycles.  The chip's power leaves it 1.5 to 1.8 GHz meanwhile.  Two chunks of 2048 behind 28001 keys, 16 heads of 64, fp16:
// 557 us, 818 TFLOP/s (a plain product of 8192 x 8192 x 8192 1140); 16384 tokens, window 2048, 32 heads of 128, bf16: 552 us, 935 TFLOP/s (1180); 16 prompts of 587:
// 31 us (1216 workgroups, 768 of them at once).  Slower were: eight wavefronts of two heads whose products and exponentials take turns
// (727 us and 782 for the chunks and the window), halves of a tile with the next one's scores computed ahead (630 and 720), four wavefronts a SIMD (634 for the chunks).
//
// A row whose result is not finite is computed again by the kernel that never touches a hidden key (attend_row): 0 times NaN or infinity is what a product
// over a tile makes of a hidden one's values.
#include "attention.h"
#include "common.h"
#include "dma.h"
#include "launch.h"
#include "lds.h"

namespace mlora {

namespace {

constexpr int kWaves = 4, kRows = 32 * kWaves, kKeys = 64;
// 2^-kMoves: how far below a row's largest weight the base may lie; the weights are then at most 2^kMoves times 2^shift.
constexpr float kMoves = 8.0f;

template <typename T> struct Mma32;
template <> struct Mma32<__bf16> {
  static __device__ __forceinline__ f32x16 run(const Pack8& a, const Pack8& b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.bf, b.bf, c, 0, 0, 0); }
};
template <> struct Mma32<_Float16> {
  static __device__ __forceinline__ f32x16 run(const Pack8& a, const Pack8& b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.hf, b.hf, c, 0, 0, 0); }
};
template <> struct Mma32<float> {  // four 32x32x2 products, product j taking element j of every lane's piece
  static __device__ __forceinline__ f32x16 run(const Pack8& a, const Pack8& b, f32x16 c) {
    f32x4 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};

template <typename T, int D> struct Shape {
  static constexpr int kRow = D * static_cast<int>(sizeof(T)), kChunks = kRow / 16;
  static constexpr int kBytes = kKeys * kRow;             // K or V of a tile
  static constexpr int kLoads = kBytes / 1024 / kWaves;   // a wavefront's share of it
  static constexpr int kRowsPerLoad = 1024 / kRow;
  static constexpr int kLds = 2 * 2 * kBytes;

  // A read of K takes the same piece of 32 rows, one of V^T 64 bytes of four rows (in fp32 128 of rows four apart).
  static __device__ __forceinline__ int k_place(int row, int chunk) { return chunk ^ (kRow == 128 ? (row >> 1) & 7 : row & 15); }
  static __device__ __forceinline__ int v_place(int row, int chunk) {
    return chunk ^ (sizeof(T) == 4 ? ((row >> 2) & 1) << 3 : kRow == 128 ? ((row >> 1) & 1) << 2 : (row & 3) << 2);
  }
};

typedef __attribute__((address_space(3))) s16x4 LdsS16x4;
__device__ __forceinline__ float other_half(float v, float* both) {  // lanes l and l + 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  *both = __uint_as_float(r[1]);
  return __uint_as_float(r[0]);
}

// What is the same in every lane, into scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long uniform(long long v) {
  return (static_cast<long long>(uniform(static_cast<int>(v >> 32))) << 32) | static_cast<uint32_t>(uniform(static_cast<int>(v)));
}

// A workgroup's four wavefronts take 32 rows of the same head each, or 1 << together heads of one key-value head with 128 >> together rows of each (above
// four heads a wavefront's 32 columns are several heads of fewer rows):
// the same products either way, but rows that see the same keys, and few of them left over where sequences are short.  16 heads of 2: 16 prompts of 587
// tokens 37.4 us against 40.5 with a head each, 64 sequences of 13 in fp32 15.7 against 26.7, two chunks of 2048 behind 28001 the same to a hundredth.
__host__ __device__ constexpr int tile_rows(int together) { return kRows >> together; }
__host__ __device__ constexpr int row_tiles(int rows, int together) { return rows > 0 ? (rows + tile_rows(together) - 1) >> (7 - together) : 0; }

// Of lane l the sum of lanes 0 .. l, by moves between lanes (a trip through LDS for each of the six steps costs a short prompt a microsecond).
__device__ __forceinline__ int upto_lane(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // from 1, 2, 4 and 8 lanes below in its row of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // a row's last lane to all of rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // lane 31 to rows 2 and 3
  return v;
}

struct RowTile {
  int sequence, start, rows;  // first query row (of q) and how many
  int position;               // of the first
  int total, key_start;
};

// A sequence of each lane: its rows begin .. end - 1 and its keys, in one trip to memory.
struct Lengths {
  int begin = 0, end = 0, total = 0, key_start = 0;
  __device__ __forceinline__ Lengths(const MloraAttentionArgs& a, int s) {
    if (s >= a.sequences) return;
    begin = clamped(a.starts[s], a.num_rows);
    end = clamped(a.starts[s + 1], a.num_rows);
    total = keys_of(a, s, &key_start);
  }
  // Tile `index` of lane `at`'s sequence `s`.
  __device__ __forceinline__ RowTile tile(int together, int at, int s, int index) const {
    const int first = __builtin_amdgcn_readlane(begin, at), last = __builtin_amdgcn_readlane(end, at);
    RowTile t;
    t.sequence = s;
    t.start = first + index * tile_rows(together);
    t.rows = last - t.start < tile_rows(together) ? last - t.start : tile_rows(together);
    t.total = __builtin_amdgcn_readlane(total, at);
    t.key_start = __builtin_amdgcn_readlane(key_start, at);
    t.position = t.total - (last - t.start);
    return t;
  }
};

// The item-th tile of the batch, of which there are `ranks`, one a list of heads; the chip holds `at_once` of all of them at a time.  By one wavefront.  The later rows of a prompt see the most keys: the last
// first.  Of more tiles than start at once those with the largest indexes start first, whatever their sequence (up to 64 of them), so that the short ones fill
// the gaps at the end: 16 prompts of 587 tokens 32.4 us, 35.0 in the order of the rows.
__device__ __forceinline__ bool find_tile(const MloraAttentionArgs& a, int together, int ranks, int at_once, int item, int lane, RowTile* t) {
  Lengths of(a, lane);
  int mine = row_tiles(of.end - of.begin, together), upto = upto_lane(mine), tiles = __builtin_amdgcn_readlane(upto, 63);
  if (a.sequences > 64) {
    int all = mine;
    for (int s = lane + 64; s < a.sequences; s += 64) all += row_tiles(clamped(a.starts[s + 1], a.num_rows) - clamped(a.starts[s], a.num_rows), together);
    tiles = __builtin_amdgcn_readlane(upto_lane(all), 63);
  }
  if (item >= tiles) return false;
  if (static_cast<long long>(tiles) * ranks > at_once && a.sequences > 1 && a.sequences <= 64) {
    // the largest index that more than `item` tiles reach: `reached` of them lie behind it
    int index = 0, over = 1, reached = 0;
    while (__any(mine > over)) over *= 2;
    while (over - index > 1) {
      const int middle = (index + over) >> 1, of_lane = mine > middle ? mine - middle : 0, count = __builtin_amdgcn_readlane(upto_lane(of_lane), 63);
      if (count > item) {
        index = middle;
      } else {
        over = middle;
        reached = count;
      }
    }
    const unsigned long long have = __ballot(mine > index);
    const int rank = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(have >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(have), 0));
    const int at = __builtin_ctzll(__ballot((have >> lane & 1) && rank == item - reached));
    *t = of.tile(together, at, at, index);
    return true;
  }
  item = tiles - 1 - item;
  int before = 0;
  for (int base = 0; base < a.sequences; base += 64) {
    if (base) {
      of = Lengths(a, base + lane);
      mine = row_tiles(of.end - of.begin, together);
      upto = upto_lane(mine);
    }
    const unsigned long long behind = __ballot(before + upto > item);
    if (behind) {
      const int at = __builtin_ctzll(behind), index = item - (before + __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(mine, at));
      *t = of.tile(together, at, base + at, index);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// How many tiles of keys the rows of a tile see: [0, first) and [low, high), both from whole tiles of keys on.
struct KeyTiles {
  int high, low, first_tiles, count;
  __device__ __forceinline__ KeyTiles(const MloraAttentionArgs& a, int position, int rows, int total) {
    const Visible of_first = visible_keys(a, position, total), of_last = visible_keys(a, position + rows - 1, total);
    high = of_last.high;
    low = of_first.low / kKeys * kKeys;
    first_tiles = ((a.sinks < low ? a.sinks : low) + kKeys - 1) / kKeys;
    count = first_tiles + (high > low ? (high - low + kKeys - 1) / kKeys : 0);
  }
};

// Few tiles of rows with many keys (a chunk of a prompt behind a long cache) leave compute units idle, or busy for a second round that few take part
// in.  Their work is then one list: the tiles of keys of the first tile of rows, of the second and so on.  Every workgroup takes an equal share of the list, whatever rows it falls on.
// A tile of rows that lies in several shares is joined by a second launch from what each of them left in the workspace.
// A share is 32 tiles of keys at least: below it what is left and joined costs more than the balance gives.  Where so few tiles of rows are there that they leave most compute
// units idle, shares go down to `least`, if the longest tile of rows (or, of up to twice as many, the average) is longer than that by what the second launch costs (`join`): in 16 bits a tile of keys takes
// two thirds of a microsecond, in fp32 four to eight.  16 tokens of 4 prompts behind 2000 each 28 us (51 with shares of 32), 300 behind 1700 27 (34), 173 in fp32 behind 8450, 8 heads of 128, 83 (288);
// 2000 tokens by themselves would take 44, without shares 35.
// On both sides of the lines, one chunk of T tokens behind C, 16 heads of 2 of 64, us without shares / with the short ones / with shares of 32.
//   bf16 (T / 8 workgroups without shares).  The join, T = 128, C = 250, 500, 1000: 16 / 22 / 55, 21 / 23 / 56, 32 / 27 / 53.  `few`, T = 1024, C = 100, 500, 1000: 27 / 33 / 80, 35 / 36 / 61,
//   45 / 40 / 60.  Twice `few`, T = 2048, C = 100, 1000, 8000: 44 / 44 / 84, 63 / 54 / 68, 198 / 129 / 131; T = 2560: 54 / 52 / 86, 68 / 61 / 71, 182 / 136 / 137.  What the lines take is within
//   16 % of the best of the three, and 21 % off at T = 1024, C = 250 (too early) and at T = 2560, C below 1000 (too late).
//   fp32.  The join, T = 32, C = 100, 250, 500: 21 / 22 / 24, 34 / 24 / 38, 56 / 25 / 60 (too late by a third at C = 250).  `few`, T = 4096, C = 500: 465 / 362 / 361; T = 5000: 558 / 488 / 490.
constexpr int kLeastShare = 32;
struct ShareCosts {
  int few, least, join;  // few: workgroups without shares
};
__host__ __device__ constexpr ShareCosts share_costs(int dtype) { return dtype == MLORA_DTYPE_F32 ? ShareCosts{512, 2, 4} : ShareCosts{128, 4, 16}; }

// The tiles of rows of a batch of at most 64 sequences, one a lane.
struct RowTiles {
  int begin, end, total, key_start, upto;  // of this lane's sequence; upto: tiles of rows up to its end
  int tiles;                               // of rows, all of them
  int together;
  __device__ __forceinline__ RowTile tile(int r) const {  // r may differ from lane to lane
    int at = 0;  // the first sequence that ends behind r
#pragma unroll
    for (int step = 32; step >= 1; step >>= 1)
      if (__shfl(upto, at + step - 1, kWave) <= r) at += step;
    const int first = __shfl(begin, at, kWave), last = __shfl(end, at, kWave), seq_upto = __shfl(upto, at, kWave);
    RowTile t;
    t.sequence = at;
    t.total = __shfl(total, at, kWave);
    t.key_start = __shfl(key_start, at, kWave);
    t.start = first + (r - seq_upto + row_tiles(last - first, together)) * tile_rows(together);
    t.rows = last - t.start < tile_rows(together) ? last - t.start : tile_rows(together);
    t.position = t.total - (last - t.start);
    return t;
  }
  // (rows without a key count for one, so that somebody comes by and writes them)
  __device__ __forceinline__ long long units_of(const MloraAttentionArgs& a, int r) const {
    const RowTile t = tile(r < tiles ? r : tiles - 1);
    const int count = KeyTiles(a, t.position, t.rows, t.total).count;
    return r >= tiles ? 0 : count > 0 ? count : 1;
  }
  __device__ __forceinline__ RowTiles(const MloraAttentionArgs& a, int heads_together, int lane) : together(heads_together) {
    begin = end = total = key_start = 0;
    if (lane < a.sequences) {
      begin = clamped(a.starts[lane], a.num_rows);
      end = clamped(a.starts[lane + 1], a.num_rows);
      total = keys_of(a, lane, &key_start);
    }
    upto = upto_lane(row_tiles(end - begin, together));
    tiles = __builtin_amdgcn_readlane(upto, 63);
  }
};

struct Shares : RowTiles {
  long long units, per;  // tiles of keys, all of them and a share's; per = 0: not shared out
  __device__ __forceinline__ Shares(const MloraAttentionArgs& a, int shares, int together, int ranks, int lane) : RowTiles(a, together, lane) {
    units = per = 0;
    if (tiles == 0) return;
    int longest = 0;
    for (int base = 0; base < tiles; base += 64) {
      const int mine = static_cast<int>(units_of(a, base + lane));
      units += mine;
      longest = mine > longest ? mine : longest;
    }
    for (int o = 32; o >= 1; o >>= 1) {
      units += __shfl_xor(units, o, kWave);
      const int other = __shfl_xor(longest, o, kWave);
      longest = other > longest ? other : longest;
    }
    per = (units + shares - 1) / shares;
    const ShareCosts costs = share_costs(a.dtype);
    const long long alone = static_cast<long long>(tiles) * ranks, short_share = per < costs.least ? costs.least : per;  // alone: workgroups without shares
    if (alone <= costs.few ? longest >= short_share + costs.join : alone <= 2 * costs.few && units >= (short_share + costs.join) * tiles) per = short_share;
    else if (alone <= costs.few) per = 0;
    else if (per < kLeastShare) per = units > static_cast<long long>(kLeastShare) * tiles ? kLeastShare : 0;
    // (more tiles than the workspace has places for: starts that run backwards, whose sequences lie on one another)
    if (tiles >= 4 * shares || tiles > a.num_rows / tile_rows(together) + a.sequences) per = 0;
  }
  // The tile of rows that holds `unit` and the unit that it starts with.
  __device__ __forceinline__ int find(const MloraAttentionArgs& a, long long unit, int lane, long long* first) const {
    long long before = 0;
    for (int base = 0; base < tiles; base += 64) {
      const long long mine = units_of(a, base + lane);
      long long last = mine;
      for (int o = 1; o < 64; o <<= 1) {
        const long long other = __shfl_up(last, o, kWave);
        if (lane >= o) last += other;
      }
      const unsigned long long behind = __ballot(before + last > unit);
      if (behind) {
        const int at = __builtin_ctzll(behind);
        *first = before + __shfl(last - mine, at, kWave);
        return base + at;
      }
      before += __shfl(last, 63, kWave);
    }
    return -1;
  }
};

// Workspace: how many tiles of rows are shared out, what the join has to know of each, and of every (share, which end of it, head) the
// rows' (m, l), then their o.  A share has two unfinished tiles of rows at most: place 0 for one that began in front of it, place 1 for one that
// begins in it.
struct Joint {
  int share, parts, sequence, start, rows, position, total, key_start;
};
struct Unfinished {
  float2* sums;
  float* outputs;
};
__host__ __device__ inline int64_t joints_bytes(int64_t tiles) { return 16 + tiles * static_cast<int64_t>(sizeof(Joint)); }
__device__ __forceinline__ int32_t* shared_tiles(const MloraAttentionArgs& a) { return static_cast<int32_t*>(a.workspace); }
__device__ __forceinline__ Joint* joint(const MloraAttentionArgs& a, int tile) { return reinterpret_cast<Joint*>(static_cast<char*>(a.workspace) + 16) + tile; }
__device__ __forceinline__ Unfinished unfinished(const MloraAttentionArgs& a, int shares, int together, int share, int place, int rank, int dim) {
  const int ranks = a.heads >> together;
  const int64_t at = (static_cast<int64_t>(share) * 2 + place) * ranks + rank, all = static_cast<int64_t>(shares) * 2 * ranks;
  float2* const sums = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + joints_bytes(a.num_rows / tile_rows(together) + a.sequences));
  return {sums + at * kRows, reinterpret_cast<float*>(sums + all * kRows) + at * kRows * dim};
}

// The kernel's first argument where the launch left it.
__device__ __forceinline__ const MloraAttentionArgs* arguments_again() {
  uint64_t p = (uint64_t)(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(p));
  return reinterpret_cast<const MloraAttentionArgs*>(p);
}

// Workgroups that a compute unit holds at once, by the bytes of a head.
constexpr int per_unit(int row) { return row == 128 ? 3 : row == 256 ? 2 : 1; }

// What the host works out for the workgroups, which would divide for it one by one in front of their first load.
struct Grid {
  int shares, together, group;
  uint32_t kv_heads_inverse;  // 2^31 / kv_heads rounded up: right for ranks up to 2^15
  uint32_t page_inverse;      // 2^(31 + page_shift) / page rounded up, 2^page_shift <= page: key / page is (2 key page_inverse >> 32) >> page_shift for keys up to 2^29
  int page_shift;
};
constexpr int kMostHeads = 1 << 15, kItemsPerPlane = 1 << 15;

// Where keys lie: packed, in pages that hold whole tiles, in pages that hold the rows of whole loads (two chunks of 2048 behind 28001 keys in pages of 16: 613 us,
// 663 as in any pages, 575 in pages of 256 on the same machine), in any pages.
constexpr int kPacked = 0, kWholePages = 1, kLoadPages = 2, kAnyPages = 3;

template <typename T, int D, int kWhere>
__global__ __launch_bounds__(kWaves * 64, per_unit(sizeof(T) * D)) void prompt_kernel(MloraAttentionArgs a, Grid grid) {
  using S = Shape<T, D>;
  constexpr int kSteps = S::kChunks / 2, kBlocks = D / 32;
  // fp16: weights are held 2^7 times as large, so that those of 2^-21 are still normal numbers and the largest (2^15) finite
  constexpr float kShift = __is_same(T, _Float16) ? 7.0f : 0.0f;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, column = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int shares = grid.shares, together = grid.together;
  // (workgroups of one key-value head go to the same XCDs: workgroup i runs on XCD i % 8)
  const int ranks = gridDim.x, rank = blockIdx.x, item = blockIdx.y + kItemsPerPlane * blockIdx.z;
  const int of_group = static_cast<int>(__umulhi(2u * rank, grid.kv_heads_inverse)), kv_head = rank - of_group * a.kv_heads;
  // a wavefront's columns: rows row_of_wave .. + row_mask of 32 / (row_mask + 1) heads from first_head on
  const int heads_of_wave = together > 2 ? together - 2 : 0, row_mask = 31 >> heads_of_wave;
  const int first_head = kv_head * grid.group + (of_group << together) + ((wave & ((1 << together) - 1)) << heads_of_wave);
  const int row_of_wave = 32 * (wave >> together);
  RowTile tile;
  bool shared = false;
  // Of a share: tiles of keys that are left of it, and the first of them in its tile of rows.
  int left = 0, from = 0, tile_number = 0;
  long long a_share = 0;
  if (shares) {
    const Shares s(a, shares, together, ranks, lane);
    const long long per = uniform(s.per), units = uniform(s.units), unit = item * per;
    if (rank == 0 && item == 0 && threadIdx.x == 0) *shared_tiles(a) = per ? s.tiles : 0;
    if (per) {
      a_share = per;
      if (item >= shares || unit >= units) return;
      shared = true;
      long long first;
      tile_number = uniform(s.find(a, unit, lane, &first));
      from = static_cast<int>(unit - uniform(first));
      left = static_cast<int>(unit + per < units ? per : units - unit);
    }
  }
  if (!shared && !uniform(find_tile(a, together, ranks, 256 * per_unit(sizeof(T) * D), item, lane, &tile))) return;
  for (;;) {
  if (shared) tile = RowTiles(a, together, lane).tile(tile_number);
  const int sequence = uniform(tile.sequence), start = uniform(tile.start), rows = uniform(tile.rows), position = uniform(tile.position);
  const int total = uniform(tile.total), key_begin = uniform(tile.key_start);
  const KeyTiles of_rows(a, position, rows, total);
  const int high = of_rows.high, low = of_rows.low, first_tiles = of_rows.first_tiles;
  // the tiles of keys from .. to of them are this workgroup's
  const int to = shared && left < of_rows.count - from ? from + left : of_rows.count;

  // This lane's query row; rows behind the last repeat it and are not written.
  const int mine = row_of_wave + (column & row_mask);
  const int row = start + (mine < rows ? mine : rows - 1);
  const int place = position + (mine < rows ? mine : rows - 1);
  const int wave_rows = rows - row_of_wave < row_mask + 1 ? rows - row_of_wave : row_mask + 1;  // (may be negative)
  const int wave_first = position + row_of_wave, wave_last = wave_first + wave_rows - 1;
  const float scale = __builtin_fabsf(a.scale) * kLog2e;

  Pack8 query[kSteps];
  {
    const char* q = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + row * a.q_row + (first_head + (column >> (5 - heads_of_wave))) * a.q_head);
    const uint32_t turn = a.scale < 0 ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      query[s].raw = load128(q + 16 * (half + 2 * s));
#pragma unroll
      for (int d = 0; d < 4; ++d) query[s].u[d] ^= turn;
    }
  }

  f32x16 o[kBlocks];
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[d][j] = 0.0f;
  float m = -__builtin_inff(), l = 0.0f;

  const uint32_t ring_at = __builtin_amdgcn_readfirstlane(lds_address(lds));
  const int32_t* table = a.block_tables + (kWhere == kPacked ? 0 : sequence * a.table_row);
  int batch = -64, ids = 0;  // page ids batch .. batch + 63, one a lane
  unsigned long long known_pages = 0;  // which of them are pages of the cache
  int page = 0, in_page = 0;
  auto key_of = [&](int t) { return t < first_tiles ? t * kKeys : low + (t - first_tiles) * kKeys; };
  auto stage_of = [&](int t) { return (t & 1) * 2 * S::kBytes; };

  // Byte offsets of what a lane asks for in a whole tile.
  uint32_t k_offset[S::kLoads], v_offset[S::kLoads];
  const uint32_t k_row = static_cast<uint32_t>(a.k_row * sizeof(T)), v_row = static_cast<uint32_t>(a.v_row * sizeof(T));
#pragma unroll
  for (int i = 0; i < S::kLoads; ++i) {
    const int r = (wave * S::kLoads + i) * S::kRowsPerLoad + lane / S::kChunks, piece = lane % S::kChunks;
    const int from_base = kWhere == kLoadPages ? lane / S::kChunks : r;
    k_offset[i] = from_base * k_row + 16 * S::k_place(r, piece);
    v_offset[i] = from_base * v_row + 16 * S::v_place(r, piece);
  }

  // Asks for this wavefront's quarter of tile t; returns which of the tile's keys there are.
  auto request = [&](int t) -> unsigned long long {
    const int key0 = key_of(t), there = high - key0 < kKeys ? high - key0 : kKeys;
    unsigned long long valid = there == kKeys ? ~0ull : (1ull << there) - 1;
    const uint32_t k_to = ring_at + stage_of(t) + wave * S::kLoads * 1024, v_to = k_to + S::kBytes;
    if constexpr (kWhere == kLoadPages) {
      auto page_of = [&](int key) { return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(key), grid.page_inverse) >> grid.page_shift); };
      const int first = page_of(key0), last = page_of(key0 + there - 1);
      if (first < batch || last >= batch + 64) {
        batch = first;
        const int p = batch + lane;
        ids = table[p < a.table_width ? p : a.table_width - 1];
        known_pages = __ballot(ids >= 0 && ids < a.num_blocks);
      }
      const unsigned long long wanted = ((1ull << (last - first + 1)) - 1) << (first - batch);  // (nine pages at most)
      if ((known_pages & wanted) != wanted) valid &= __ballot(known_pages >> (page_of(key0 + (lane < there ? lane : there - 1)) - batch) & 1);
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int r = (wave * S::kLoads + i) * S::kRowsPerLoad, end = (there - 1) / S::kRowsPerLoad * S::kRowsPerLoad, row = r < end ? r : end;
        const int page = page_of(key0 + row), in_page = key0 + row - page * a.page;
        const int64_t block = known_pages >> (page - batch) & 1 ? __builtin_amdgcn_readlane(ids, page - batch) : 0;  // (what lies in a page of no cache is masked)
        const char* const k = uniform(reinterpret_cast<const char*>(static_cast<const T*>(a.k) + block * a.k_block + in_page * a.k_row + kv_head * a.k_head));
        const char* const v = uniform(reinterpret_cast<const char*>(static_cast<const T*>(a.v) + block * a.v_block + in_page * a.v_row + kv_head * a.v_head));
        const int behind = row + lane / S::kChunks - (there - 1);
        const uint32_t back = behind > 0 ? behind : 0;  // (a place behind the last key repeats it)
        dma16_from(k, k_offset[i] - back * k_row, k_to + i * 1024);
        dma16_from(v, v_offset[i] - back * v_row, v_to + i * 1024);
      }
    } else if constexpr (kWhere != kAnyPages) {
      const char *k, *v;
      if constexpr (kWhere == kPacked) {
        k = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + (static_cast<int64_t>(key_begin) + key0) * a.k_row + kv_head * a.k_head);
        v = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + (static_cast<int64_t>(key_begin) + key0) * a.v_row + kv_head * a.v_head);
      } else {
        // (a tile lies behind the one asked for before it, but where the first keys end and the last begin)
        in_page += kKeys;
        if (t == from || t == first_tiles) {
          page = key0 / a.page;
          in_page = key0 - page * a.page;
        } else if (in_page >= a.page) {
          ++page;
          in_page = 0;
        }
        if (page < batch || page >= batch + 64) {
          batch = page;
          const int p = batch + lane;
          ids = table[p < a.table_width ? p : a.table_width - 1];
        }
        const int id = __builtin_amdgcn_readlane(ids, page - batch);
        if (id < 0 || id >= a.num_blocks) return 0;  // (the stage keeps what it held: every key of it is masked)
        k = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + id * a.k_block + in_page * a.k_row + kv_head * a.k_head);
        v = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + id * a.v_block + in_page * a.v_row + kv_head * a.v_head);
      }
      k = uniform(k);
      v = uniform(v);
      if (there == kKeys) {
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
          dma16_from(k, k_offset[i], k_to + i * 1024);
          dma16_from(v, v_offset[i], v_to + i * 1024);
        }
      } else {
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
          const int r = (wave * S::kLoads + i) * S::kRowsPerLoad + lane / S::kChunks;
          const uint32_t back = r < there ? 0 : r - there + 1;  // (a place behind the last key repeats it)
          dma16_from(k, k_offset[i] - back * k_row, k_to + i * 1024);
          dma16_from(v, v_offset[i] - back * v_row, v_to + i * 1024);
        }
      }
    } else {
      const int key = key0 + (lane < there ? lane : there - 1), page0 = key0 / a.page, of_page = key / a.page;
      if (page0 < batch || (key0 + there - 1) / a.page >= batch + 64) {
        batch = page0;
        const int p = batch + lane;
        ids = table[p < a.table_width ? p : a.table_width - 1];
      }
      const int id = __shfl(ids, of_page - batch, kWave), row_of_page = key - of_page * a.page;
      const bool known = id >= 0 && id < a.num_blocks;
      valid &= __ballot(known);
      const T *k = static_cast<const T*>(a.k), *v = static_cast<const T*>(a.v);
      if (known) {  // (else the first row of the cache)
        k += id * a.k_block + row_of_page * a.k_row;
        v += id * a.v_block + row_of_page * a.v_row;
      }
      const uint64_t ka = reinterpret_cast<uintptr_t>(k + kv_head * a.k_head), va = reinterpret_cast<uintptr_t>(v + kv_head * a.v_head);
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int r = (wave * S::kLoads + i) * S::kRowsPerLoad + lane / S::kChunks, piece = lane % S::kChunks;
        const uint64_t kr = __shfl(static_cast<unsigned long long>(ka), r, kWave), vr = __shfl(static_cast<unsigned long long>(va), r, kWave);
        dma16v(reinterpret_cast<const char*>(kr) + 16 * S::k_place(r, piece), k_to + i * 1024);
        dma16v(reinterpret_cast<const char*>(vr) + 16 * S::v_place(r, piece), v_to + i * 1024);
      }
    }
    return valid;
  };

  // The tiles that this wavefront's rows see end here; the others are only asked for.
  const int seen_end = a.causal ? (wave_last < high - 1 ? wave_last : high - 1) : high - 1;  // their last key
  int own = wave_rows <= 0 || seen_end < 0 ? 0 : seen_end < low ? first_tiles : first_tiles + (seen_end - low) / kKeys + 1;
  own = own < to ? own : to;

  const int i16 = lane & 15;
  unsigned long long next_valid = from < to ? request(from) : 0;
  for (int t = from; t < to; ++t) {
    const int key0 = key_of(t);
    const unsigned long long valid = next_valid;
    wait_loads<0>();
    stage_barrier();  // this tile is there, and the one before it has been read
    if (t + 1 < to) next_valid = request(t + 1);
    if (t >= own) continue;

    const char* const k_tile = lds + stage_of(t);
    const char* const v_tile = k_tile + S::kBytes;
    f32x16 s[2];
    const bool second = key0 + 32 <= seen_end;  // (fp32, where a block of 32 keys costs 2048 cycles for each product: 64 sequences of 13 tokens 13.9 us, 15.7 without)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[b][j] = 0.0f;
      if (sizeof(T) == 4 && b == 1 && !second) continue;
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        Pack8 key;
        key.raw = load128(k_tile + (32 * b + column) * S::kRow + 16 * S::k_place(32 * b + column, half + 2 * st));
        s[b] = Mma32<T>::run(key, query[st], s[b]);
      }
    }
    if constexpr (sizeof(T) == 4) asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(s[0]), "+v"(s[1]));  // (the branch over the masks below)
    __builtin_amdgcn_s_setprio(0);
    const bool all_behind = !a.causal || key0 + kKeys - 1 <= wave_first;
    const bool all_near = !a.window || key0 > wave_last - a.window || key0 + kKeys <= a.sinks;
    if (!(all_behind && all_near && valid == ~0ull)) {
      // key 32 b + 8 (j / 4) + 4 half + j % 4 of the tile
      const int behind = (a.causal ? place : INT32_MAX / 2) - key0 - 4 * half;
      const int far = a.window ? place - a.window - key0 - 4 * half : INT32_MIN / 2;
      const int sinks = a.window ? a.sinks - key0 - 4 * half : 0;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t known = static_cast<uint32_t>(valid >> (32 * b)) >> (4 * half);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int of_block = 8 * (j >> 2) + (j & 3), e = 32 * b + of_block;
          const bool seen = (e <= behind) & ((e > far) | (e < sinks)) & ((known >> of_block & 1) != 0);
          s[b][j] = seen ? s[b][j] : -__builtin_inff();
        }
      }
    }
    float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(fmaxf(top, s[0][j]), s[1][j]);
    float upper;
    const float lower = other_half(top, &upper);
    top = fmaxf(lower, upper) * scale;
    if (__any(top > m + kMoves)) {
      const float moved = fmaxf(m, top);
      const float alpha = moved == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - moved);
      m = moved;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[d][j] *= alpha;
    }
    const float base = (m == -__builtin_inff() ? 0.0f : m) - kShift;
    // V^T of 16 keys, at head size 128 read one step ahead of its product: a transposing read takes some 400 cycles when every wavefront reads, and two
    // wavefronts a SIMD hide less of it than three (16384 tokens of 32 heads 567 us against 586; at head size 64, 2 x 2048 tokens behind 28001, 574 against 568).
    constexpr bool kAhead = D == 128;
    union Piece { s16x4 part[2]; Pack8 all; };
    Piece v[2][kBlocks];
    auto read_v = [&](int step, Piece* to) {
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 16 * step + 8 * e + 4 * half + (i16 >> 2);
          const int chunk = 4 * d + 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
          to[d].part[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(v_tile + r * S::kRow + 16 * S::v_place(r, chunk) + 8 * (i16 & 1)));
        }
    };
    if constexpr (sizeof(T) == 2 && kAhead) read_v(0, v[0]);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j) s[b][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j], scale, -base));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if constexpr (sizeof(T) == 2) {
        Pack8 ones;
        const float one[8] = {1, 1, 1, 1, 1, 1, 1, 1};
        pack8<T>(one, ones);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!kAhead) read_v(2 * b + c, v[c]);
          else if (2 * b + c < 3) read_v(2 * b + c + 1, v[1 - c]);
          float w8[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w8[j] = s[b][8 * c + j];
          Pack8 weights;
          // (the matrix cores take weights of the element type, half a step of it off each: as two pieces of 16 bits they would cost this product, half of
          // all of them, twice; the rounded weights' sum is what the outputs are divided by)
          pack8<T>(w8, weights);
          l = dot8<T>(weights, ones, l);
#pragma unroll
          for (int d = 0; d < kBlocks; ++d) o[d] = Mma32<T>::run(v[c][d].all, weights, o[d]);
        }
      } else {
        if (b == 1 && !second) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          l += s[b][j];
          const int r = 32 * b + 8 * (j >> 2) + 4 * half + (j & 3);
#pragma unroll
          for (int d = 0; d < kBlocks; ++d) {
            const float v = *reinterpret_cast<const float*>(v_tile + r * S::kRow + 16 * S::v_place(r, 8 * d + (column >> 2)) + 4 * (column & 3));
            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[b][j], o[d], 0, 0, 0);
          }
        }
      }
    }
  }
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(o[d]));  // (the loop may end right behind a product)
  {
    float upper;
    const float lower = other_half(l, &upper);
    l = lower + upper;
  }
  // (the arguments once more from memory: held over the loop they would take the scalar registers that it needs)
  const MloraAttentionArgs& args = *arguments_again();
  if (shared && rank == 0 && from == 0 && threadIdx.x == 0) {
    const long long behind = of_rows.count - left;  // tiles of keys in the shares behind this one
    const int parts = behind > 0 ? 1 + static_cast<int>((behind + a_share - 1) / a_share) : 1;
    *joint(args, tile_number) = {item, parts, sequence, start, rows, position, total, key_begin};
  }
  if (shared && to - from < of_rows.count) {  // for the join
    const Unfinished u = unfinished(args, shares, together, item, from ? 0 : 1, rank, D);
    const int at = 32 * wave + column;
    if (half == 0) u.sums[at] = make_float2(m, l);
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int p = 0; p < 4; ++p)
        *reinterpret_cast<f32x4*>(u.outputs + at * D + 32 * d + 8 * p + 4 * half) = f32x4{o[d][4 * p], o[d][4 * p + 1], o[d][4 * p + 2], o[d][4 * p + 3]};
    __syncthreads();  // (the stages have been read)
  } else {
  // (also a row without a visible key, 0 / 0)
  const float inverse = 1.0f / l;
  bool finite = true;
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      o[d][j] *= inverse;
      finite &= __builtin_fabsf(o[d][j]) < __builtin_inff();
    }
  unsigned long long again = __ballot(!finite && mine < rows);
  again = (again | again >> 32) & 0xffffffffull;
  if (mine < rows && !(again >> column & 1)) {
    T* out = static_cast<T*>(args.out) + row * args.out_row + (first_head + (column >> (5 - heads_of_wave))) * args.out_head;
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) {
      if constexpr (sizeof(T) == 2) {
        // halves exchange so that a lane has eight elements side by side: of group 2 p the lower, of 2 p + 1 the upper
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float w8[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w8[j] = o[d][8 * p + j];
          Pack8 w, x;
          pack8<T>(w8, w);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const auto r = __builtin_amdgcn_permlane32_swap(w.u[j], w.u[2 + j], false, false);
            x.u[j] = r[0];
            x.u[2 + j] = r[1];
          }
          store128(out + 32 * d + 16 * p + 8 * half, x.raw);
        }
      } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) *reinterpret_cast<f32x4*>(out + 32 * d + 8 * p + 4 * half) = f32x4{o[d][4 * p], o[d][4 * p + 1], o[d][4 * p + 2], o[d][4 * p + 3]};
      }
    }
  }
  __syncthreads();  // (the stages have been read)
  while (again) {
    const int c = __builtin_ctzll(again);
    again &= again - 1;
    const int r = c & row_mask;
    const Place at{sequence, total, key_begin, wave_first + r};
    attend_row<T>(args, at, start + row_of_wave + r, first_head + (c >> (5 - heads_of_wave)), lane, reinterpret_cast<float*>(lds) + wave * MLORA_MAX_HEAD_DIM);
  }
  if (shared) __syncthreads();
  }
  left -= of_rows.count ? to - from : 1;
  if (!shared || left <= 0) return;
  from = 0;
  ++tile_number;
  }
}

// Joins the parts of 32 rows of a tile that lies in several shares, eight rows a wavefront.
template <typename T, int D>
__global__ __launch_bounds__(256) void prompt_join_kernel(MloraAttentionArgs a, int shares, int together) {
  constexpr int kPer = D / 64, kOwn = 8;
  __shared__ float scratch[kWaves][MLORA_MAX_HEAD_DIM];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rank = blockIdx.y, number = blockIdx.x >> 2;
  if (number >= *shared_tiles(a)) return;
  const Joint t = *joint(a, number);
  const int of_wave = blockIdx.x & 3, group = a.heads / a.kv_heads;  // (the wavefront that had them)
  const int heads_of_wave = together > 2 ? together - 2 : 0, row_mask = 31 >> heads_of_wave;
  const int first_head = rank % a.kv_heads * group + ((rank / a.kv_heads) << together) + ((of_wave & ((1 << together) - 1)) << heads_of_wave);
  const int column = kOwn * wave, row_of_wave = 32 * (of_wave >> together), first_left = 32 * of_wave + column;  // columns from `column` on
  if (t.parts < 2 || row_of_wave + (column & row_mask) >= t.rows) return;
  const int own = first_left + (lane & (kOwn - 1));  // the row whose (m, l) this lane looks after
  float most = -__builtin_inff(), sum = 0.0f, x[kOwn][kPer] = {};
#pragma unroll 4
  for (int p = 0; p < t.parts; ++p) most = fmaxf(most, unfinished(a, shares, together, t.share + p, p ? 0 : 1, rank, D).sums[own].x);
  constexpr int kAtOnce = 4;  // parts whose outputs are on their way together
  for (int base = 0; base < t.parts; base += kAtOnce) {
    float factor[kAtOnce], v[kAtOnce][kOwn][kPer];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int p = base + j < t.parts ? base + j : t.parts - 1;
      const Unfinished u = unfinished(a, shares, together, t.share + p, p ? 0 : 1, rank, D);
      const float2 ml = u.sums[own];
      factor[j] = base + j >= t.parts ? 0.0f : ml.x == most ? 1.0f : __builtin_amdgcn_exp2f(ml.x - most);
      sum += base + j >= t.parts ? 0.0f : factor[j] * ml.y;
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[j][i][e] = u.outputs[(first_left + i) * D + 64 * e + lane];
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (base + j >= t.parts) break;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const float f = __shfl(factor[j], i, kWave);
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[i][e] += f * v[j][i][e];
      }
    }
  }
  unsigned again = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int r = row_of_wave + ((column + i) & row_mask), head = first_head + ((column + i) >> (5 - heads_of_wave));
    const float l = __shfl(sum, i, kWave);
    bool finite = true;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      x[i][e] /= l;
      finite &= __builtin_fabsf(x[i][e]) < __builtin_inff();
    }
    if (r >= t.rows) continue;
    if (!__all(finite)) {
      again |= 1u << i;
      continue;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) static_cast<T*>(a.out)[(t.start + r) * a.out_row + head * a.out_head + 64 * e + lane] = from_f32<T>(x[i][e]);
  }
  for (; again; again &= again - 1) {
    const int c = column + __builtin_ctz(again), r = row_of_wave + (c & row_mask);
    attend_row<T>(a, Place{t.sequence, t.total, t.key_start, t.position + r}, t.start + r, first_head + (c >> (5 - heads_of_wave)), lane, scratch[wave]);
  }
}

// At least four lists of shares are left where there are many rows, so that a list is not long for those who look for their place in it.
int heads_together(const MloraAttentionArgs& a) {
  const int group = a.heads / a.kv_heads, rows = a.num_rows / a.sequences;
  int together = group % 4 == 0 && a.heads >= 16 ? 2 : group % 2 == 0 && a.heads >= 8 ? 1 : 0;
  // Sequences of few rows fill a tile with as many heads as there are, up to 32, and so read their keys once: 233 rows of 42 sequences behind 63560 keys each,
  // 8 heads of one of 64, 183 us, 393 in tiles of two heads; 64 sequences of 13 tokens in fp32 12.1 us, 13.9 in tiles of four.
  for (int more = together + 1; more <= 5 && group % (1 << more) == 0; ++more)
    if (rows <= tile_rows(more)) together = more;
  return together;
}

// Shares of a list: as many workgroups as the chip holds at once.
int shares_of(const MloraAttentionArgs& a) {
  const int resident = 256 * per_unit(a.dim * (a.dtype == MLORA_DTYPE_F32 ? 4 : 2)) / (a.heads >> heads_together(a));
  return resident > 1 ? resident : 1;
}

template <typename T, int D> int launch(const MloraAttentionArgs& a) {
  const int where = !a.block_tables ? kPacked : a.page % kKeys == 0 ? kWholePages : a.page % Shape<T, D>::kRowsPerLoad == 0 && a.page >= 8 ? kLoadPages : kAnyPages;
  const int together = heads_together(a);
  const long long items = a.num_rows / tile_rows(together) + a.sequences;  // at most that many tiles of rows
  const int shares = prompt_workspace_bytes(&a) && a.workspace && a.workspace_bytes >= static_cast<int64_t>(prompt_workspace_bytes(&a)) ? shares_of(a) : 0;
  const long long all = items > shares ? items : shares;
  const dim3 grid(a.heads >> together, static_cast<unsigned>(all < kItemsPerPlane ? all : kItemsPerPlane), static_cast<unsigned>((all + kItemsPerPlane - 1) / kItemsPerPlane));
  const int page = a.block_tables ? a.page : 1, page_shift = 31 - __builtin_clz(static_cast<uint32_t>(page));
  const Grid given{shares, together, a.heads / a.kv_heads, static_cast<uint32_t>(((1ll << 31) + a.kv_heads - 1) / a.kv_heads),
                   static_cast<uint32_t>(((1ull << (31 + page_shift)) + page - 1) / page), page_shift};
  constexpr int kLds = Shape<T, D>::kLds;
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  if (where == kPacked) {
    allow_lds<prompt_kernel<T, D, kPacked>>(kLds);
    prompt_kernel<T, D, kPacked><<<grid, kWaves * 64, kLds, stream>>>(a, given);
  } else if (where == kWholePages) {
    allow_lds<prompt_kernel<T, D, kWholePages>>(kLds);
    prompt_kernel<T, D, kWholePages><<<grid, kWaves * 64, kLds, stream>>>(a, given);
  } else if (where == kLoadPages) {
    allow_lds<prompt_kernel<T, D, kLoadPages>>(kLds);
    prompt_kernel<T, D, kLoadPages><<<grid, kWaves * 64, kLds, stream>>>(a, given);
  } else {
    allow_lds<prompt_kernel<T, D, kAnyPages>>(kLds);
    prompt_kernel<T, D, kAnyPages><<<grid, kWaves * 64, kLds, stream>>>(a, given);
  }
  const int rc = check_launch("mlora_prompt_attention");
  if (rc || !shares) return rc;
  prompt_join_kernel<T, D><<<dim3(static_cast<unsigned>(4 * items), a.heads >> together), 256, 0, stream>>>(a, shares, together);
  return check_launch("mlora_prompt_attention (join)");
}

}  // namespace

bool prompt_supported(const MloraAttentionArgs* a) {
  if ((a->dim != 64 && a->dim != 128) || !attention_vectors_ok(a)) return false;
  if (a->block_tables ? a->table_width < 1 || a->num_blocks < 1 : a->num_keys < 1) return false;
  // a tile's rows are reached by 32-bit offsets from its first
  const int64_t most = INT32_MAX / (kKeys * 4);
  if (a->k_row < 0 || a->v_row < 0 || a->k_row > most || a->v_row > most) return false;
  const int64_t items = static_cast<int64_t>(a->num_rows / tile_rows(heads_together(*a))) + a->sequences;
  return a->heads <= kMostHeads && items <= static_cast<int64_t>(kItemsPerPlane) * 65535 && 4 * items <= INT32_MAX;
}

// Scratch of the shares where the work may be shared out: few tiles of rows for the chip, and enough keys to share.
size_t prompt_workspace_bytes(const MloraAttentionArgs* a) {
  if (!prompt_supported(a) || a->sequences > 64 || a->heads > 512) return 0;
  const ShareCosts costs = share_costs(a->dtype);
  const int64_t shares = shares_of(*a), tiles = a->num_rows / tile_rows(heads_together(*a)) + a->sequences;
  // As the device will decide, with the longest that a sequence may be, or of packed keys the average (the rows of a prompt by itself see half of its keys each): the
  // launch that joins costs one also where it finds nothing to do.
  const int64_t there = a->block_tables ? static_cast<int64_t>(a->table_width) * a->page : a->num_keys / a->sequences;
  const int64_t near = a->window ? static_cast<int64_t>(a->window) + a->sinks + kRows + 2 * kKeys : INT64_MAX, keys = there < near ? there : near;
  const bool by_itself = !a->block_tables && !a->key_starts && a->causal;
  const int64_t least = tiles * (a->heads >> heads_together(*a)) <= costs.few * (by_itself ? 1 : 2) ? costs.least + costs.join : by_itself ? 2 * kLeastShare : kLeastShare;
  if (tiles >= (a->block_tables ? 2 : 1) * shares || keys <= least * kKeys) return 0;
  return static_cast<size_t>(joints_bytes(tiles) + shares * 2 * (a->heads >> heads_together(*a)) * kRows * (8 + 4 * a->dim));
}

int launch_prompt(const MloraAttentionArgs* a) {
  if (a->dim == 64) {
    if (a->dtype == MLORA_DTYPE_BF16) return launch<__bf16, 64>(*a);
    return a->dtype == MLORA_DTYPE_F16 ? launch<_Float16, 64>(*a) : launch<float, 64>(*a);
  }
  if (a->dtype == MLORA_DTYPE_BF16) return launch<__bf16, 128>(*a);
  return a->dtype == MLORA_DTYPE_F16 ? launch<_Float16, 128>(*a) : launch<float, 128>(*a);
}

}  // namespace mlora
