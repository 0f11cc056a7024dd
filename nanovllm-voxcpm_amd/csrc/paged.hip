// Attention of one new token per sequence over a paged cache, head sizes 64 and 128 (mlora_decode_attention).
//
// Bound by memory: every visible key and value is read once, and 16 heads of a group meet it on the matrix cores at a
// thousandth of their rate.  So the kernel is laid out for bytes in flight.  A workgroup takes a run of tiles of one
// sequence and key-value head, its wavefronts equal pieces of the run; a wavefront asks for its tiles' rows by direct loads into a ring
// of its own in LDS and waits for nobody else until the sums meet.  Rows lie in the ring with their 16-byte pieces exchanged (piece ^ f(row)), so that the
// reads below meet every bank once.  Scores come out of the first product with the keys along the registers and the heads along the lanes (K Q^T),
// which is how the second one (V^T P^T) wants its weights: they pass from one to the other in registers.  V^T is read through the
// transposing LDS read.
//
// Few long sequences are split: the tiles of the whole batch are shared out in parts of one size, as many as fill the chip, whatever sequence
// they belong to.  Workgroups find their part from context_lens alone.  A sequence of one part is written straight away; the others leave (m, l, o) per
// head in the workspace, and a second launch joins them: o = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m), in the order of the parts.
// 3 sequences of up to 131072 keys, 32 heads, 8 of 128, bf16: 225 us, 5.3 TB/s (a large copy 5.2); 208 sequences, window 1024, 16 heads,
// 2 of 64: 23 us, 4.5 TB/s; 64 of up to 2048: 13.3 us, 2.6 TB/s (bound by the trips to memory that the longest one's wavefronts make one behind the other).
#include "attention.h"
#include "common.h"
#include "dma.h"
#include "launch.h"
#include "lds.h"

namespace mlora {

namespace {

constexpr int kBlockHeads = 16;
constexpr int kWorkgroups = 512;  // that a batch is cut into: two a compute unit
constexpr int kLongWhole = 128;   // tiles of a sequence that four wavefronts take by themselves

// What a hidden key's row is read from.
__device__ __align__(16) uint32_t zero_row[MLORA_MAX_HEAD_DIM];

template <typename T, int D, int W> struct Shape {
  static constexpr int kWaves = W, kStages = W == 4 ? 2 : 1;
  static constexpr int kRow = D * static_cast<int>(sizeof(T)), kChunks = kRow / 16;
  static constexpr int kKeys = sizeof(T) == 2 ? 32 : 16;  // one contraction of the second product
  static constexpr int kBytes = kKeys * kRow, kLoads = kBytes / 1024, kRowsPerLoad = 1024 / kRow;
  static constexpr int kRing = kWaves * kStages * 2 * kBytes, kLds = kRing + kWaves * kBlockHeads * 8 + kBlockHeads * 8 + kWaves * 4;
  static_assert(kWaves * kBlockHeads * (D + 4) * 4 <= kRing, "the outputs meet where the rings were");
  // (K: 16 rows' piece of the same number in one read; V: 8 rows' pairs of pieces, in fp32 4 rows' four)
  static __device__ __forceinline__ int k_place(int row, int chunk) { return chunk ^ (kRow == 128 ? (row >> 1) & 7 : row & 15); }
  static __device__ __forceinline__ int v_place(int row, int chunk) {
    return chunk ^ (sizeof(T) == 4 ? ((row >> 2) & 3) << 2 : kRow == 128 ? ((row >> 1) & 3) << 1 : (row & 7) << 1);
  }
};

typedef __attribute__((address_space(3))) s16x4 LdsS16x4;

// Over the lanes of the same number modulo 16.
template <typename F> __device__ __forceinline__ float over_groups(float v, F f) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float group_max(float v) { return over_groups(v, [](float x, float y) { return fmaxf(x, y); }); }
__device__ __forceinline__ float group_sum(float v) { return over_groups(v, [](float x, float y) { return x + y; }); }

// The tiles of a sequence: those of the first keys, then those of the last.
template <int KEYS> struct Tiles {
  Visible seen;
  int first_tiles, low_tile, count;
  __device__ __forceinline__ Tiles(const MloraAttentionArgs& a, int total) {
    seen = visible_keys(a, total - 1, total);
    first_tiles = (seen.first + KEYS - 1) / KEYS;
    low_tile = seen.low / KEYS;
    count = first_tiles + (seen.high > seen.low ? (seen.high + KEYS - 1) / KEYS - low_tile : 0);
  }
  __device__ __forceinline__ int key(int tile) const { return (tile < first_tiles ? tile : tile - first_tiles + low_tile) * KEYS; }
  __device__ __forceinline__ bool sees_all(int tile, int key0) const {
    return tile < first_tiles ? key0 + KEYS <= seen.first : key0 >= seen.low && key0 + KEYS <= seen.high;
  }
  __device__ __forceinline__ bool sees(int tile, int key) const { return tile < first_tiles ? key < seen.first : key >= seen.low && key < seen.high; }
};

struct Part {
  int sequence, index, parts, tiles_per_part;
};

// Inclusive sums over the lanes: within rows of 16 by shifts, then the rows' last lanes to the rows behind them.
template <int kControl, int kRows> __device__ __forceinline__ uint32_t plus_moved(uint32_t v) {
  return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, kRows, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = plus_moved<0x111, 0xf>(v);
  v = plus_moved<0x112, 0xf>(v);
  v = plus_moved<0x114, 0xf>(v);
  v = plus_moved<0x118, 0xf>(v);
  v = plus_moved<0x142, 0xa>(v);
  return plus_moved<0x143, 0xc>(v);
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)); }

// Part number `item` of the batch; `target`: parts to cut the batch's tiles into (0: one a sequence).  By one wavefront.
template <int KEYS, int kWaves> __device__ __forceinline__ bool find_part(const MloraAttentionArgs& a, int item, int target, int lane, Part* p) {
  if (!target) {
    *p = {item, 0, 1, INT32_MAX};
    return item < a.sequences;
  }
  int key_start;
  uint32_t mine = 0;
  uint64_t tiles = 0;
  for (int base = 0; base < a.sequences; base += 64) {
    mine = base + lane < a.sequences ? Tiles<KEYS>(a, keys_of(a, base + lane, &key_start)).count : 0;
    tiles += lane_value(wave_scan(mine), 63);
  }
  // (whole rounds of the wavefronts)
  const uint64_t least = (tiles + target - 1) / target;
  const uint32_t per = static_cast<uint32_t>(least + kWaves - 1) / kWaves * kWaves + (least == 0 ? kWaves : 0);
  uint32_t before = 0;
  for (int base = 0; base < a.sequences; base += 64) {
    const int s = base + lane;
    if (a.sequences > 64) mine = s < a.sequences ? Tiles<KEYS>(a, keys_of(a, s, &key_start)).count : 0;
    const uint32_t parts = s < a.sequences ? (mine + per - 1) / per + (mine == 0) : 0, upto = wave_scan(parts);
    const unsigned long long behind = __ballot(before + upto > static_cast<uint32_t>(item));
    if (behind) {
      const int at = __builtin_ctzll(behind);
      p->sequence = base + at;
      p->parts = lane_value(parts, at);
      p->index = item - (before + lane_value(upto, at) - p->parts);
      p->tiles_per_part = per;
      return true;
    }
    before += lane_value(upto, 63);
  }
  return false;
}

// Workspace: {first part, parts} of every sequence, (m, l) of every part and head, o of every part and head.
struct Workspace {
  int32_t* rows;
  float2* sums;
  float* outputs;
};
__host__ __device__ inline int64_t workspace_rows_bytes(int sequences) { return (static_cast<int64_t>(sequences) * 8 + 15) & ~15ll; }
__device__ __forceinline__ Workspace workspace_of(const MloraAttentionArgs& a, int items) {
  char* p = static_cast<char*>(a.workspace);
  Workspace w;
  w.rows = reinterpret_cast<int32_t*>(p);
  w.sums = reinterpret_cast<float2*>(p + workspace_rows_bytes(a.sequences));
  w.outputs = reinterpret_cast<float*>(w.sums + ((static_cast<int64_t>(items) * a.heads + 1) & ~1ll));
  return w;
}

// `group`: heads of a key-value head; `pages`: log2 of the page where it is a power of two of 8 rows or more and rows lie near enough for 32-bit offsets, else -1.
template <typename T, int D, int W>
__global__ __launch_bounds__(W * 64, W == 4 ? 2 : 1) void paged_kernel(MloraAttentionArgs a, int target, int pages, int group) {
  using S = Shape<T, D, W>;
  constexpr int kWaves = W, kStages = S::kStages;
  constexpr int kKeys = S::kKeys, kSteps = S::kChunks / 4, kBlocks = D / 16;
  // fp16: weights, at most 1, are held 2^15 times as large: the largest is finite, those of 2^-29 are still normal numbers
  constexpr float kShift = __is_same(T, _Float16) ? 15.0f : 0.0f;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, column = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv_head = blockIdx.y, head_block = blockIdx.z;
  const int head_in_group = head_block * kBlockHeads + column;
  const bool real = head_in_group < group;
  const int head = kv_head * group + (real ? head_in_group : 0);

  // What the first trip to memory can bring: lengths and, where the sequence is known without them, its queries and first page ids.
  Pack8 query[kSteps];
  int batch = 0, ids = 0;  // page ids batch .. batch + 63, one a lane
  auto load_query = [&](int sequence) {
    const char* q = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + sequence * a.q_row + head * a.q_head);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) query[s].raw = load128(q + 16 * (g + 4 * s));
  };
  auto load_ids = [&](int sequence, int page) {
    batch = page;
    const int p = batch + lane;
    ids = a.block_tables[sequence * a.table_row + (p < a.table_width ? p : a.table_width - 1)];
  };
  if (!target) {
    load_ids(blockIdx.x, 0);
    load_query(blockIdx.x);
  }
  Part part;
  if (!__builtin_amdgcn_readfirstlane(find_part<kKeys, kWaves>(a, blockIdx.x, target, lane, &part))) return;
  const int sequence = __builtin_amdgcn_readfirstlane(part.sequence);
  int key_start;
  const Tiles<kKeys> tiles(a, __builtin_amdgcn_readfirstlane(keys_of(a, sequence, &key_start)));
  const int per = __builtin_amdgcn_readfirstlane(part.tiles_per_part), index = __builtin_amdgcn_readfirstlane(part.index);
  const int begin = index * per;  // (index is 0 where `per` is the largest number)
  const int end = tiles.count - begin < per ? tiles.count : begin + per;
  // this wavefront's run
  const int share = (end - begin + kWaves - 1) / kWaves;
  const int from = begin + wave * share, to = from + share < end ? from + share : end;
  const int working = share ? (end - begin + share - 1) / share : 0;  // wavefronts that have one
  const float scale = a.scale * kLog2e;

  f32x4 o[kBlocks];
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) o[d] = f32x4{0, 0, 0, 0};
  float m = -__builtin_inff(), l = 0.0f;
  bool any = false;

  if (from < to) {
    auto page_of = [&](int key) { return pages >= 0 ? key >> pages : key / a.page; };
    if (target) {
      load_ids(sequence, page_of(tiles.key(from)));
      load_query(sequence);
    }
    if (!real) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) query[s].raw = i32x4{0, 0, 0, 0};
    }
    unsigned long long known = __ballot(ids >= 0 && ids < a.num_blocks);
    char* const ring = lds + wave * (kStages * 2 * S::kBytes);
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane(lds_address(ring));
    uint32_t masks[kStages];
    const int own_row = lane / S::kChunks, piece = lane % S::kChunks;
    const uint32_t k_from = own_row * static_cast<uint32_t>(a.k_row * sizeof(T)), v_from = own_row * static_cast<uint32_t>(a.v_row * sizeof(T));
    uint32_t k_offset[S::kLoads], v_offset[S::kLoads];  // of a lane's pieces in a tile that lies in one page
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int r = i * S::kRowsPerLoad + own_row;
      k_offset[i] = r * static_cast<uint32_t>(a.k_row * sizeof(T)) + 16 * S::k_place(r, piece);
      v_offset[i] = r * static_cast<uint32_t>(a.v_row * sizeof(T)) + 16 * S::v_place(r, piece);
    }

    // Asks for the rows of tile t.
    auto request = [&](int t, int stage) {
      const int key0 = tiles.key(t), page0 = page_of(key0), last = page_of(key0 + kKeys - 1);
      if (page0 < batch || last >= batch + 64) {
        load_ids(sequence, page0);
        known = __ballot(ids >= 0 && ids < a.num_blocks);
      }
      const unsigned long long wanted = ((last - page0 == 63 ? 0ull : 1ull << (last - page0 + 1)) - 1) << (page0 - batch);
      const uint32_t to_k = ring_at + stage * 2 * S::kBytes, to_v = to_k + S::kBytes;
      if (pages >= 0 && tiles.sees_all(t, key0) && (known & wanted) == wanted) {
        masks[stage] = kKeys == 32 ? 0xffffffffu : 0xffffu;
        if ((1 << pages) >= kKeys) {  // all rows lie in one page (an address each instead of one a load: 64 streams of up to 2048 keys 13.3 us, 15.2 before)
          const int id = __builtin_amdgcn_readlane(ids, page0 - batch), in_page = key0 & ((1 << pages) - 1);
          const char* const k = uniform(reinterpret_cast<const char*>(static_cast<const T*>(a.k) + id * a.k_block + in_page * a.k_row + kv_head * a.k_head));
          const char* const v = uniform(reinterpret_cast<const char*>(static_cast<const T*>(a.v) + id * a.v_block + in_page * a.v_row + kv_head * a.v_head));
#pragma unroll
          for (int i = 0; i < S::kLoads; ++i) {
            dma16_from(k, k_offset[i], to_k + i * 1024);
            dma16_from(v, v_offset[i], to_v + i * 1024);
          }
          return;
        }
        // the rows of one load lie in one page
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
          const int key = key0 + i * S::kRowsPerLoad, id = __builtin_amdgcn_readlane(ids, (key >> pages) - batch), in_page = key & ((1 << pages) - 1);
          const char* k = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + id * a.k_block + in_page * a.k_row + kv_head * a.k_head);
          const char* v = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + id * a.v_block + in_page * a.v_row + kv_head * a.v_head);
          const int r = i * S::kRowsPerLoad + own_row;
          dma16_from(uniform(k), k_from + 16 * S::k_place(r, piece), to_k + i * 1024);
          dma16_from(uniform(v), v_from + 16 * S::v_place(r, piece), to_v + i * 1024);
        }
        return;
      }
      // Row by row: lanes 0 .. 31 find the keys', lanes 32 .. 63 the values'.
      const int key = key0 + (lane & 31), page = page_of(key);
      const int id = __shfl(ids, page - batch, kWave);
      const bool valid = (lane & 31) < kKeys && tiles.sees(t, key) && id >= 0 && id < a.num_blocks;
      masks[stage] = static_cast<uint32_t>(__ballot(valid));
      const int64_t in_page = key - page * a.page;
      const bool is_v = lane >= 32;
      const char* row = reinterpret_cast<const char*>(
          is_v ? static_cast<const T*>(a.v) + id * a.v_block + in_page * a.v_row + kv_head * a.v_head
               : static_cast<const T*>(a.k) + id * a.k_block + in_page * a.k_row + kv_head * a.k_head);
      if (!valid) row = reinterpret_cast<const char*>(zero_row);
      const uint32_t lo = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)), hi = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) >> 32);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
          const int r = i * S::kRowsPerLoad + own_row, chunk = kv ? S::v_place(r, piece) : S::k_place(r, piece);
          const uint32_t l32 = __shfl(lo, 32 * kv + r, kWave), h32 = __shfl(hi, 32 * kv + r, kWave);
          const char* p = reinterpret_cast<const char*>((static_cast<uint64_t>(h32) << 32) | l32) + 16 * chunk;
          dma16v(p, (kv ? to_v : to_k) + i * 1024);
        }
      }
    };

#pragma unroll
    for (int i = 0; i < kStages; ++i)
      if (from + i < to) request(from + i, i);
    for (int t = from; t < to; ++t) {
      const int stage = kStages == 1 ? 0 : (t - from) & 1;
      if (kStages == 2 && t + 1 < to) wait_loads<2 * S::kLoads>();
      else wait_loads<0>();
      const char* const k_tile = ring + stage * 2 * S::kBytes;
      const char* const v_tile = k_tile + S::kBytes;
      const uint32_t mask = masks[stage];
      float s[kKeys / 4];
#pragma unroll
      for (int b = 0; b < kKeys / 16; ++b) {
        f32x4 products[1] = {{0, 0, 0, 0}};
        f32x4& c = products[0];
        const int r = 16 * b + column;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          Pack8 key;
          key.raw = load128(k_tile + r * S::kRow + 16 * S::k_place(r, g + 4 * st));
          c = Mma<T>::run(key, query[st], c);
        }
        if constexpr (sizeof(T) == 4) mfma_settle(products);  // (the branch over the masks below)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * b + j] = c[j] * scale;
      }
      any |= mask != 0;
      if (mask != (kKeys == 32 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
        for (int b = 0; b < kKeys / 16; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!(mask >> (16 * b + 4 * g + j) & 1)) s[4 * b + j] = -__builtin_inff();
      }
      float top = s[0];
#pragma unroll
      for (int j = 1; j < kKeys / 4; ++j) top = fmaxf(top, s[j]);
      top = fmaxf(m, group_max(top));
      const float bottom = top == -__builtin_inff() ? 0.0f : top, base = bottom - kShift;
      const float alpha = __builtin_amdgcn_exp2f(m - bottom);
      m = top;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][j] *= alpha;
#pragma unroll
      for (int j = 0; j < kKeys / 4; ++j) s[j] = __builtin_amdgcn_exp2f(s[j] - base);
      if constexpr (sizeof(T) == 2) {
        // The matrix cores take weights of the element type, half a step of it off each.  The sum is of the rounded ones, so that what is left out of the
        // numerator is left out of the denominator too: equal values come out as they are.  (Held as two pieces of 16 bits, weights would be as good
        // as fp32: an error against 64 bits of 0.0017 in bf16, of which the output's own rounding is 0.0016, in place of 0.0019; 1 stream 7.85 us and 64 streams 12.41,
        // as they are 7.64 and 12.26.)
        float p8[8];
        const float one[8] = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
        for (int j = 0; j < 8; ++j) p8[j] = s[j];
        Pack8 weights, ones;
        pack8<T>(p8, weights);
        pack8<T>(one, ones);
        l = dot8<T>(weights, ones, l);
        const int i = column;
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) {
          union { s16x4 half[2]; Pack8 all; } v;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int r = 16 * b + 4 * g + (i >> 2);
            const char* p = v_tile + r * S::kRow + 16 * S::v_place(r, 2 * d + ((i & 3) >> 1)) + 8 * (i & 1);
            v.half[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS16x4*)(p));
          }
          o[d] = Mma<T>::run(v.all, weights, o[d]);
        }
      } else {
        const int i = column;
#pragma unroll
        for (int j = 0; j < 4; ++j) l += s[j];
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = 4 * g + j;
            const float v = *reinterpret_cast<const float*>(v_tile + r * S::kRow + 16 * S::v_place(r, 4 * d + (i >> 2)) + 4 * (i & 3));
            o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s[j], o[d], 0, 0, 0);
          }
        }
      }
      if (t + kStages < to) {
        wait_lds();  // (every read of this stage has come back)
        request(t + kStages, stage);
      }
    }
#pragma unroll
    for (int d = 0; d < kBlocks; d += 4) mfma_settle(*reinterpret_cast<f32x4(*)[4]>(&o[d]));
  }

  // The wavefronts' sums meet: every one weighs its own to the common maximum, then the outputs are added up element by element.
  float2* const shared_ml = reinterpret_cast<float2*>(lds + S::kRing);  // [wave][head]
  float2* const shared_sum = shared_ml + kWaves * kBlockHeads;          // [head]
  int* const shared_any = reinterpret_cast<int*>(shared_sum + kBlockHeads);
  l = group_sum(l);
  if (g == 0) shared_ml[wave * kBlockHeads + column] = make_float2(m, l);
  if (lane == 0) shared_any[wave] = any;
  __syncthreads();  // (the rings have been read, too)
  float* const shared_o = reinterpret_cast<float*>(lds);  // [wave][head][D + 4]
  if (wave < working) {
    // (each group of lanes looks at a quarter of the wavefronts)
    float most = -__builtin_inff(), sum = 0.0f;
    float2 ml[kWaves / 4];
#pragma unroll
    for (int i = 0; i < kWaves / 4; ++i) {
      const int v = 4 * i + g;
      ml[i] = v < working ? shared_ml[v * kBlockHeads + column] : make_float2(-__builtin_inff(), 0.0f);
      most = fmaxf(most, ml[i].x);
    }
    most = group_max(most);
#pragma unroll
    for (int i = 0; i < kWaves / 4; ++i) sum += ml[i].y * (ml[i].x == most ? 1.0f : __builtin_amdgcn_exp2f(ml[i].x - most));
    sum = group_sum(sum);
    const float factor = m == most ? 1.0f : __builtin_amdgcn_exp2f(m - most);
    if (real) {
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) *reinterpret_cast<f32x4*>(shared_o + (wave * kBlockHeads + column) * (D + 4) + 16 * d + 4 * g) = o[d] * factor;
    }
    if (wave == 0 && g == 0) shared_sum[column] = make_float2(most, sum);
  }
  const bool some = __any(lane < working && shared_any[lane < kWaves ? lane : 0]);
  __syncthreads();

  const int items = gridDim.x;
  const bool whole = part.parts == 1;
  const Workspace w = workspace_of(a, items);
  if (target && threadIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && index == 0) {
    w.rows[2 * sequence] = blockIdx.x;
    w.rows[2 * sequence + 1] = part.parts;
  }
#pragma unroll
  for (int i = threadIdx.x; i < kBlockHeads * D; i += kWaves * 64) {
    const int row = i / D, e = i % D, out_in_group = head_block * kBlockHeads + row;
    if (out_in_group >= group) break;
    const int out_head = kv_head * group + out_in_group;
    float x = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v)
      if (v < working) x += shared_o[(v * kBlockHeads + row) * (D + 4) + e];
    const float2 ml = some ? shared_sum[row] : make_float2(-__builtin_inff(), -1.0f);
    if (whole) {
      static_cast<T*>(a.out)[sequence * a.out_row + out_head * a.out_head + e] = from_f32<T>(some ? x / ml.y : 0.0f);
    } else {
      const int64_t at = static_cast<int64_t>(blockIdx.x) * a.heads + out_head;
      if (e == 0) w.sums[at] = ml;
      w.outputs[at * D + e] = x;
    }
  }
}

// Joins the parts of a (sequence, head): their weights to the common maximum first, kJoinParts of them at a time.
constexpr int kJoinParts = 256;
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(MloraAttentionArgs a, int items) {
  constexpr int kRuns = 256 / D;  // threads of an element, each with every kRuns-th part
  __shared__ float tops[4], sums[4], factors[kJoinParts], values[kRuns][D];
  const int sequence = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Workspace w = workspace_of(a, items);
  const int first = w.rows[2 * sequence], parts = w.rows[2 * sequence + 1];
  if (parts < 2) return;
  const float2* const at = w.sums + static_cast<int64_t>(first) * a.heads + head;
  const float* const from = w.outputs + (static_cast<int64_t>(first) * a.heads + head) * D;
  const int64_t stride = static_cast<int64_t>(a.heads) * D;
  float most = -__builtin_inff();
  for (int i = threadIdx.x; i < parts; i += 256) {
    const float2 ml = at[static_cast<int64_t>(i) * a.heads];
    if (!(ml.y < 0)) most = fmaxf(most, ml.x);
  }
  most = wave_max(most);
  if (lane == 0) tops[wave] = most;
  __syncthreads();
  most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const int run = threadIdx.x / D, e = threadIdx.x - run * D;
  float sum = 0, x = 0;
  bool some = false;
  for (int base = 0; base < parts; base += kJoinParts) {
    const int n = parts - base < kJoinParts ? parts - base : kJoinParts;
    float factor = 0.0f;
    if (static_cast<int>(threadIdx.x) < n) {
      const float2 ml = at[static_cast<int64_t>(base + threadIdx.x) * a.heads];
      if (!(ml.y < 0)) {  // (a part that saw no key counts for nothing)
        some = true;
        factor = ml.x == most ? 1.0f : __builtin_amdgcn_exp2f(ml.x - most);
        sum += factor * ml.y;
      }
    }
    if (base) __syncthreads();
    factors[threadIdx.x] = factor;
    __syncthreads();
    int i = run;
    for (; i + 7 * kRuns < n; i += 8 * kRuns) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = from[(base + i + j * kRuns) * stride + e];
#pragma unroll
      for (int j = 0; j < 8; ++j) x += factors[i + j * kRuns] * v[j];
    }
    for (; i < n; i += kRuns) x += factors[i] * from[(base + i) * stride + e];
  }
  values[run][e] = x;
  sum = wave_sum(sum);
  some = __any(some);
  if (lane == 0) sums[wave] = some ? sum : -1.0f;
  __syncthreads();
  if (run) return;
  sum = 0, x = 0, some = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (sums[i] < 0) continue;
    some = true;
    sum += sums[i];
  }
#pragma unroll
  for (int i = 0; i < kRuns; ++i) x += values[i][e];
  static_cast<T*>(a.out)[sequence * a.out_row + head * a.out_head + e] = from_f32<T>(some ? x / sum : 0.0f);
}

int units_of_part(int heads, int kv_heads) { return kv_heads * ((heads / kv_heads + kBlockHeads - 1) / kBlockHeads); }
// Wavefronts of a workgroup where a few of them have to take a whole sequence.
constexpr int wide(int dim) { return dim == 64 ? 16 : 8; }

// How a call is cut.  Every way is right for every length; the lengths themselves only the device knows.
//   Many sequences and heads (or a window, which bounds what a sequence costs): a workgroup of four wavefronts each, no join.
//   Few, and none longer than four tiles a wavefront of the wide workgroups: one of these each, no join.
//   Else the batch's tiles are shared out in parts of four wavefronts and joined.
// us by the device's clock, four wavefronts whole / wide workgroups / parts.  208 sequences, 2 heads of 64, window 1024: 23 / 27 / 40; 3 of up to 131072, 8 heads of 128:
// 1475 / 1400 / 224.  On both sides of the lines, sequences of up to `longest` keys, 2 heads of 64, in tables as wide as the longest:
//   units (sequences times heads)  128 | 160 | 192 | 256 | 384 at 1000 keys: 11.2 / 9.7 / 12.9 | 11.7 / 10.0 / 16.4 | 12.0 / 10.7 / 16.6 | 12.6 / 11.5 / 20.7 | 15.2 / 18.5 / 26.4
//   (the wide ones would be faster by 9 to 14 % up to 256 units, and slower by a fifth at 384);
//   64 tiles, 2000 | 4000 keys of 16 sequences 16.5 / 12.1 / 11.5 and 28 / 17.6 / 13.6, of 64 17.4 / 13.5 / 17.2 and 28 / 21 / 22, of 80 at 4000 29 / 23 / 30;
//   kLongWhole, 4000 | 8000 keys of 128 sequences 32 / 30 / 36 and 67 / 70 / 72, of 32 28 / 18 / 16 and 50 / 31 / 22.
// A table wider than the longest sequence is cut for its width: 64 streams of up to 2048 keys 12.9 us, 15.8 in tables of 9 pages of 256 and more.
struct Way {
  int waves, target;  // target: parts wanted, 0: none
};
Way cut_of(const MloraAttentionArgs& a) {
  const int units = units_of_part(a.heads, a.kv_heads);
  const int64_t keys = a.dtype == MLORA_DTYPE_F32 ? 16 : 32, most_keys = static_cast<int64_t>(a.table_width) * a.page;
  const int64_t seen = a.window ? static_cast<int64_t>(a.window) + a.sinks + 2 * keys : INT64_MAX, tiles = ((most_keys < seen ? most_keys : seen) + keys - 1) / keys;
  if (static_cast<int64_t>(a.sequences) * units >= 192 && tiles <= kLongWhole) return {4, 0};
  if (tiles <= 4 * wide(a.dim)) return {wide(a.dim), 0};
  return {4, (kWorkgroups + units - 1) / units};
}

template <typename T, int D, int W> int launch(const MloraAttentionArgs& a, int target, int pages) {
  using S = Shape<T, D, W>;
  const int items = a.sequences + target;
  allow_lds<paged_kernel<T, D, W>>(S::kLds);
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  const int group = a.heads / a.kv_heads;
  paged_kernel<T, D, W><<<dim3(items, a.kv_heads, (group + kBlockHeads - 1) / kBlockHeads), W * 64, S::kLds, stream>>>(a, target, pages, group);
  if (const int rc = check_launch("mlora_decode_attention")) return rc;
  if (!target) return 0;
  join_kernel<T, D><<<dim3(a.sequences, a.heads), 256, 0, stream>>>(a, items);
  return check_launch("mlora_decode_attention (join)");
}

template <typename T, int D> int launch_shape(const MloraAttentionArgs& a) {
  Way cut = cut_of(a);
  if (!a.workspace || a.workspace_bytes < static_cast<int64_t>(paged_workspace_bytes(&a))) cut.target = 0;
  int pages = -1;
  const int64_t most = INT32_MAX / (32 * 4);
  if (a.page >= 8 && (a.page & (a.page - 1)) == 0 && a.k_row >= 0 && a.v_row >= 0 && a.k_row <= most && a.v_row <= most) pages = __builtin_ctz(a.page);
  return cut.waves == 4 ? launch<T, D, 4>(a, cut.target, pages) : launch<T, D, wide(D)>(a, cut.target, pages);
}

}  // namespace

bool paged_supported(const MloraAttentionArgs* a) {
  if ((a->dim != 64 && a->dim != 128) || !attention_vectors_ok(a) || a->table_width < 1 || units_of_part(a->heads, a->kv_heads) > 65535 || a->heads > 65535) return false;
  // a dimension of a launch has fewer than 2^32 threads
  const Way cut = cut_of(*a);
  return (static_cast<int64_t>(a->sequences) + cut.target) * cut.waves * 64 <= UINT32_MAX;
}

size_t paged_workspace_bytes(const MloraAttentionArgs* a) {
  const Way cut = cut_of(*a);
  if (!cut.target) return 0;
  const int64_t items = static_cast<int64_t>(a->sequences) + cut.target;
  return static_cast<size_t>(workspace_rows_bytes(a->sequences) + ((items * a->heads + 1) & ~1ll) * 8 + items * a->heads * a->dim * 4);
}

int launch_paged(const MloraAttentionArgs* a) {
  if (a->dim == 64) {
    if (a->dtype == MLORA_DTYPE_BF16) return launch_shape<__bf16, 64>(*a);
    return a->dtype == MLORA_DTYPE_F16 ? launch_shape<_Float16, 64>(*a) : launch_shape<float, 64>(*a);
  }
  if (a->dtype == MLORA_DTYPE_BF16) return launch_shape<__bf16, 128>(*a);
  return a->dtype == MLORA_DTYPE_F16 ? launch_shape<_Float16, 128>(*a) : launch_shape<float, 128>(*a);
}

}  // namespace mlora
