// Attention of one new token per sequence over a paged cache, head sizes 64 and 128 (mlora_decode_attention).
//
// Bound by memory: every visible key and value is read once, and 16 heads of a group meet it on the matrix cores at a
// thousandth of their rate.  So the kernel is laid out for bytes in flight.  A workgroup takes a run of tiles of one
// sequence and key-value head, its four wavefronts a quarter of the run each; a wavefront asks for its tiles' rows by direct loads into a ring
// of its own in LDS, two stages deep, and waits for nobody else.  Rows lie in the ring with their 16-byte pieces exchanged (piece ^ f(row)), so that the
// reads below meet every bank once.  Scores come out of the first product with the keys along the registers and the heads along the lanes (K Q^T),
// which is how the second one (V^T P^T) wants its weights: they pass from one to the other in registers.  V^T is read through the
// transposing LDS read.
//
// The length is split: the tiles of the whole batch are shared out in parts of one size, as many as fill the chip, whatever sequence
// they belong to.  Workgroups find their part from context_lens alone.  A sequence of one part is written straight away; the others leave (m, l, o) per
// head in the workspace, and a second launch joins them: o = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m), in the order of the parts.
#include "attention.h"
#include "common.h"
#include "dma.h"
#include "launch.h"
#include "lds.h"

namespace mlora {

namespace {

constexpr int kWaves = 4, kStages = 2, kBlockHeads = 16;
// Parts that a batch is cut into: workgroups of about two rounds over the chip, two workgroups a compute unit.
constexpr int kWorkgroups = 1024;

// What a hidden key's row is read from.
__device__ __align__(16) uint32_t zero_row[MLORA_MAX_HEAD_DIM];

template <typename T, int D> struct Shape {
  static constexpr int kRow = D * static_cast<int>(sizeof(T)), kChunks = kRow / 16;
  static constexpr int kKeys = sizeof(T) == 2 ? 32 : 16;  // one contraction of the second product
  static constexpr int kBytes = kKeys * kRow, kLoads = kBytes / 1024, kRowsPerLoad = 1024 / kRow;
  static constexpr int kLds = kWaves * kStages * 2 * kBytes;
  // (K: 16 rows' piece of the same number in one read; V: 8 rows' pairs of pieces, in fp32 4 rows' four)
  static __device__ __forceinline__ int k_place(int row, int chunk) { return chunk ^ (kRow == 128 ? (row >> 1) & 7 : row & 15); }
  static __device__ __forceinline__ int v_place(int row, int chunk) {
    return chunk ^ (sizeof(T) == 4 ? ((row >> 2) & 3) << 2 : kRow == 128 ? ((row >> 1) & 3) << 1 : (row & 7) << 1);
  }
};

typedef __attribute__((address_space(3))) s16x4 LdsS16x4;

__device__ __forceinline__ float group_max(float v) {  // over the lanes of the same number modulo 16
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float group_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

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
  __device__ __forceinline__ bool sees(int tile, int key) const { return tile < first_tiles ? key < seen.first : key >= seen.low && key < seen.high; }
};

struct Part {
  int sequence, index, parts, tiles_per_part;
};

// Part number `item` of the batch; `target`: parts to cut the batch's tiles into (0: one a sequence).  By one wavefront.
template <int KEYS> __device__ __forceinline__ bool find_part(const MloraAttentionArgs& a, int item, int target, int lane, Part* p) {
  if (!target) {
    *p = {item, 0, 1, INT32_MAX};
    return item < a.sequences;
  }
  int key_start, mine = 0;
  long long tiles = 0;
  for (int s = lane; s < a.sequences; s += 64) {
    mine = Tiles<KEYS>(a, keys_of(a, s, &key_start)).count;
    tiles += mine;
  }
  for (int o = 32; o >= 1; o >>= 1) tiles += __shfl_xor(tiles, o, kWave);
  // (never fewer than a tile a wavefront)
  int per = static_cast<int>((tiles + target - 1) / target);
  per = per < kWaves ? kWaves : per;
  int before = 0;
  for (int base = 0; base < a.sequences; base += 64) {
    const int s = base + lane;
    if (a.sequences > 64) mine = s < a.sequences ? Tiles<KEYS>(a, keys_of(a, s, &key_start)).count : 0;
    const int parts = s < a.sequences ? (mine + per - 1) / per + (mine == 0) : 0;
    int upto = parts;
    for (int o = 1; o < 64; o <<= 1) {
      const int other = __shfl_up(upto, o, kWave);
      if (lane >= o) upto += other;
    }
    const unsigned long long behind = __ballot(before + upto > item);
    if (behind) {
      const int at = __builtin_ctzll(behind);
      p->sequence = base + at;
      p->parts = __shfl(parts, at, kWave);
      p->index = item - (before + __shfl(upto, at, kWave) - p->parts);
      p->tiles_per_part = per;
      return true;
    }
    before += __shfl(upto, 63, kWave);
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

template <typename T, int D>
__global__ __launch_bounds__(kWaves * 64, 2) void paged_kernel(MloraAttentionArgs a, int target, int page_shift) {
  using S = Shape<T, D>;
  constexpr int kKeys = S::kKeys, kSteps = S::kChunks / 4, kBlocks = D / 16;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, column = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = a.heads / a.kv_heads, head_blocks = (group + kBlockHeads - 1) / kBlockHeads;
  const int kv_head = blockIdx.y / head_blocks, head_block = blockIdx.y - kv_head * head_blocks;
  Part part;
  if (!find_part<kKeys>(a, blockIdx.x, target, lane, &part)) return;
  const int sequence = __builtin_amdgcn_readfirstlane(part.sequence);
  int key_start;
  const Tiles<kKeys> tiles(a, __builtin_amdgcn_readfirstlane(keys_of(a, sequence, &key_start)));
  const int per = __builtin_amdgcn_readfirstlane(part.tiles_per_part), index = __builtin_amdgcn_readfirstlane(part.index);
  const int begin = index * per;  // (index is 0 where `per` is the largest number)
  const int end = tiles.count - begin < per ? tiles.count : begin + per;
  // this wavefront's run
  const int share = (end - begin + kWaves - 1) / kWaves;
  const int from = begin + wave * share, to = from + share < end ? from + share : end;

  const int head_in_group = head_block * kBlockHeads + column;
  const bool real = head_in_group < group;
  const int head = kv_head * group + (real ? head_in_group : 0);
  const float scale = a.scale * kLog2e;

  f32x4 o[kBlocks];
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) o[d] = f32x4{0, 0, 0, 0};
  float m = -__builtin_inff(), l = 0.0f;
  bool any = false;

  if (from < to) {
    Pack8 query[kSteps];
    const T* q = static_cast<const T*>(a.q) + sequence * a.q_row + head * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) query[s].raw = real ? load128(reinterpret_cast<const char*>(q) + 16 * (g + 4 * s)) : i32x4{0, 0, 0, 0};

    char* const ring = lds + wave * (kStages * 2 * S::kBytes);
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane(lds_address(ring));
    const int32_t* table = a.block_tables + sequence * a.table_row;
    int batch = -64, ids = 0;  // page ids batch .. batch + 63, one a lane
    uint32_t masks[kStages];

    // Asks for the rows of tile t.
    auto request = [&](int t, int stage) {
      const int key0 = tiles.key(t), key = key0 + (lane & 31);
      const int page0 = page_shift >= 0 ? key0 >> page_shift : key0 / a.page, page = page_shift >= 0 ? key >> page_shift : key / a.page;
      const int last = page_shift >= 0 ? (key0 + kKeys - 1) >> page_shift : (key0 + kKeys - 1) / a.page;
      if (page0 < batch || last >= batch + 64) {
        batch = page0;
        const int p = batch + lane;
        ids = table[p < a.table_width ? p : a.table_width - 1];
      }
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
          const int r = i * S::kRowsPerLoad + lane / S::kChunks, piece = lane % S::kChunks;
          const int chunk = kv ? S::v_place(r, piece) : S::k_place(r, piece);
          const uint32_t l32 = __shfl(lo, 32 * kv + r, kWave), h32 = __shfl(hi, 32 * kv + r, kWave);
          const char* p = reinterpret_cast<const char*>((static_cast<uint64_t>(h32) << 32) | l32) + 16 * chunk;
          dma16v(p, ring_at + (stage * 2 + kv) * S::kBytes + i * 1024);
        }
      }
    };

    request(from, 0);
    if (from + 1 < to) request(from + 1, 1);
    for (int t = from; t < to; ++t) {
      const int stage = (t - from) & 1;
      if (t + 1 < to) wait_loads<2 * S::kLoads>();
      else wait_loads<0>();
      const char* const k_tile = ring + stage * 2 * S::kBytes;
      const char* const v_tile = k_tile + S::kBytes;
      const uint32_t mask = stage ? masks[1] : masks[0];
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
      const float base = top == -__builtin_inff() ? 0.0f : top;
      const float alpha = __builtin_amdgcn_exp2f(m - base);
      m = top;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][j] *= alpha;
#pragma unroll
      for (int j = 0; j < kKeys / 4; ++j) {
        s[j] = __builtin_amdgcn_exp2f(s[j] - base);
        l += s[j];
      }
      if constexpr (sizeof(T) == 2) {
        float p8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p8[j] = s[j];
        Pack8 weights;
        pack8<T>(p8, weights);
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

  // The four wavefronts' sums: weights to the common maximum first, then element by element.
  l = group_sum(l);
  __syncthreads();  // (the rings have been read)
  float* const shared_o = reinterpret_cast<float*>(lds);  // [wave][head][D + 4]
  float* const shared_m = shared_o + kWaves * kBlockHeads * (D + 4);
  float* const shared_l = shared_m + kWaves * kBlockHeads;
  if (g == 0) {
    shared_m[wave * kBlockHeads + column] = m;
    shared_l[wave * kBlockHeads + column] = any ? l : -1.0f;  // (a wavefront that saw no key)
  }
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) *reinterpret_cast<f32x4*>(shared_o + (wave * kBlockHeads + column) * (D + 4) + 16 * d + 4 * g) = o[d];
  __syncthreads();

  const int items = gridDim.x;
  const bool whole = part.parts == 1;
  Workspace w = workspace_of(a, items);
  if (target && threadIdx.x == 0 && blockIdx.y == 0 && index == 0) {
    w.rows[2 * sequence] = blockIdx.x;
    w.rows[2 * sequence + 1] = part.parts;
  }
  constexpr int kPer = D / 16;  // elements of a thread: 16 threads a head
  const int row = threadIdx.x >> 4, e0 = (threadIdx.x & 15) * kPer;
  const int out_in_group = head_block * kBlockHeads + row;
  if (out_in_group >= group) return;
  const int out_head = kv_head * group + out_in_group;
  float most = -__builtin_inff();
  bool some = false;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    if (shared_l[v * kBlockHeads + row] < 0) continue;
    some = true;
    most = fmaxf(most, shared_m[v * kBlockHeads + row]);
  }
  float sum = 0, x[kPer] = {};
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    if (shared_l[v * kBlockHeads + row] < 0) continue;
    const float mv = shared_m[v * kBlockHeads + row], factor = mv == most ? 1.0f : __builtin_amdgcn_exp2f(mv - most);
    sum += factor * shared_l[v * kBlockHeads + row];
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] += factor * shared_o[(v * kBlockHeads + row) * (D + 4) + e0 + e];
  }
  if (whole) {
    T* out = static_cast<T*>(a.out) + sequence * a.out_row + out_head * a.out_head + e0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) out[e] = from_f32<T>(some ? x[e] / sum : 0.0f);
  } else {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * a.heads + out_head;
    if ((threadIdx.x & 15) == 0) w.sums[at] = make_float2(most, some ? sum : -1.0f);
#pragma unroll
    for (int e = 0; e < kPer; ++e) w.outputs[at * D + e0 + e] = x[e];
  }
}

// Joins the parts of a (sequence, head).
template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(MloraAttentionArgs a, int items) {
  constexpr int kRuns = 256 / D;  // threads of an element, each with every kRuns-th part
  __shared__ float tops[4], sums[kRuns], values[kRuns][D];
  const int sequence = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 63;
  const Workspace w = workspace_of(a, items);
  const int first = w.rows[2 * sequence], parts = w.rows[2 * sequence + 1];
  if (parts < 2) return;
  const float2* const at = w.sums + static_cast<int64_t>(first) * a.heads + head;
  float most = -__builtin_inff();
  for (int i = threadIdx.x; i < parts; i += 256) {
    const float2 ml = at[static_cast<int64_t>(i) * a.heads];
    if (ml.y >= 0 || ml.y != ml.y) most = fmaxf(most, ml.x);
  }
  most = wave_max(most);
  if (lane == 0) tops[threadIdx.x >> 6] = most;
  __syncthreads();
  most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const int run = threadIdx.x / D, e = threadIdx.x - run * D;
  float sum = 0, x = 0;
  bool some = false;
  for (int i = run; i < parts; i += kRuns) {
    const float2 ml = at[static_cast<int64_t>(i) * a.heads];
    if (ml.y < 0) continue;
    some = true;
    const float factor = ml.x == most ? 1.0f : __builtin_amdgcn_exp2f(ml.x - most);
    sum += factor * ml.y;
    x += factor * w.outputs[(static_cast<int64_t>(first + i) * a.heads + head) * D + e];
  }
  values[run][e] = x;
  if (e == 0) sums[run] = some ? sum : -1.0f;
  __syncthreads();
  if (run) return;
  sum = 0, x = 0, some = false;
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    if (sums[i] < 0) continue;
    some = true;
    sum += sums[i];
    x += values[i][e];
  }
  static_cast<T*>(a.out)[sequence * a.out_row + head * a.out_head + e] = from_f32<T>(some ? x / sum : 0.0f);
}

int units_of_part(int heads, int kv_heads) { return kv_heads * ((heads / kv_heads + kBlockHeads - 1) / kBlockHeads); }
int parts_wanted(int heads, int kv_heads) { return (kWorkgroups + units_of_part(heads, kv_heads) - 1) / units_of_part(heads, kv_heads); }

template <typename T, int D> int launch(const MloraAttentionArgs& a) {
  const bool split = a.workspace && a.workspace_bytes >= static_cast<int64_t>(paged_workspace_bytes(a.sequences, a.heads, a.kv_heads, a.dim));
  const int target = split ? parts_wanted(a.heads, a.kv_heads) : 0;
  const int items = a.sequences + target;
  int shift = 0;
  while ((1 << shift) < a.page && shift < 30) ++shift;
  if ((1 << shift) != a.page) shift = -1;
  constexpr int kJoin = (kWaves * kBlockHeads * (D + 4) + 2 * kWaves * kBlockHeads) * 4;
  constexpr int kLds = Shape<T, D>::kLds > kJoin ? Shape<T, D>::kLds : kJoin;
  allow_lds<paged_kernel<T, D>>(kLds);
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  paged_kernel<T, D><<<dim3(items, units_of_part(a.heads, a.kv_heads)), kWaves * 64, kLds, stream>>>(a, target, shift);
  if (const int rc = check_launch("mlora_decode_attention")) return rc;
  if (!split) return 0;
  join_kernel<T, D><<<dim3(a.sequences, a.heads), 256, 0, stream>>>(a, items);
  return check_launch("mlora_decode_attention (join)");
}

}  // namespace

bool paged_supported(const MloraAttentionArgs* a) {
  return (a->dim == 64 || a->dim == 128) && attention_vectors_ok(a) && a->table_width > 0 && units_of_part(a->heads, a->kv_heads) <= 65535 && a->heads <= 65535;
}

size_t paged_workspace_bytes(int sequences, int heads, int kv_heads, int dim) {
  const int64_t items = static_cast<int64_t>(sequences) + parts_wanted(heads, kv_heads);
  return static_cast<size_t>(workspace_rows_bytes(sequences) + ((items * heads + 1) & ~1ll) * 8 + items * heads * dim * 4);
}

int launch_paged(const MloraAttentionArgs* a) {
  if (a->dim == 64) {
    if (a->dtype == MLORA_DTYPE_BF16) return launch<__bf16, 64>(*a);
    return a->dtype == MLORA_DTYPE_F16 ? launch<_Float16, 64>(*a) : launch<float, 64>(*a);
  }
  if (a->dtype == MLORA_DTYPE_BF16) return launch<__bf16, 128>(*a);
  return a->dtype == MLORA_DTYPE_F16 ? launch<_Float16, 128>(*a) : launch<float, 128>(*a);
}

}  // namespace mlora
