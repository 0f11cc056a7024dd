// First product of the adapters beside an 8-bit linear: h[t, j] = sum_k x8[t, k] A[slot of t, j, k], for every slice (mlora_project's first launch; the row's scale
// comes with the base product's).
//
// The e4m3 numbers of x become 16-bit ones, exactly, in registers; the wavefronts of a workgroup take 64 columns of K each in turn and add up through LDS.  In front of the
// tiles' linear the rows are put in the order of their slots first, and a workgroup has 64 rows of that order, one slice, up to 64 ranks; few rows stay where they
// are, and a workgroup has the rows of one slot, which it looks for itself, one slice and 16 ranks.
#include "common.h"
#include "dma.h"
#include "launch.h"
#include "lds.h"
#include "project.h"

namespace mlora {

namespace {

// h of four ranks from j on of one row; ranks from r to `ranks` are zero.  Whether an infinity or a NaN is among them.
__device__ __forceinline__ bool store_h(const MloraProjectArgs& a, int row, int slice, int j, const f32x4& sum) {
  const int ranks = padded_ranks(a.r), width = a.num_slices * ranks;
  if (j >= ranks) return false;
  __bf16 h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(j + i < a.r ? sum[i] : 0.0f, &h[i], &l[i]);
  uint16_t* const at = intermediate(a) + static_cast<int64_t>(row) * width + slice * ranks + j;
  __builtin_memcpy(at, h, 8);
  __builtin_memcpy(at + static_cast<int64_t>(a.num_rows) * width, l, 8);
  uint32_t words[2];
  __builtin_memcpy(words, h, 8);
  return pair_beyond(words[0]) || pair_beyond(words[1]);
}

constexpr int kRowWaves = 8, kRowBatch = kRowWaves * 64;

// The rows of slot blockIdx.x, sixteen of its ranks in one slice; where that leaves compute units without work, sixteen rows in turn a workgroup (blockIdx.z).
template <typename T> __global__ __launch_bounds__(kRowWaves * 64) void shrink8_rows_kernel(MloraProjectArgs a) {
  __shared__ int32_t found[kRowBatch];
  __shared__ int counts[kRowWaves];
  __shared__ f32x4 parts[kRowWaves][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int groups = (a.r + 15) / 16, slice = blockIdx.y / groups, first = (blockIdx.y - slice * groups) * 16, slot = blockIdx.x;
  const T* const A = static_cast<const T*>(a.slices[slice].a) + (static_cast<int64_t>(slot) * a.r + (first + m < a.r ? first + m : a.r - 1)) * a.k;
  for (int base = 0; base < a.num_rows; base += kRowBatch) {
    const int t = base + static_cast<int>(threadIdx.x);
    const unsigned long long here = __ballot(t < a.num_rows && a.token_to_slot[t < a.num_rows ? t : 0] == slot);
    if (lane == 0) counts[wave] = __builtin_popcountll(here);
    __syncthreads();
    int count = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) {
      before += w < wave ? counts[w] : 0;
      count += counts[w];
    }
    if (here >> lane & 1) found[before + __builtin_popcountll(here & ((1ull << lane) - 1))] = t;
    __syncthreads();
    for (int i0 = 16 * blockIdx.z; i0 < count; i0 += 16 * gridDim.z) {
      const int row = found[i0 + m < count ? i0 + m : count - 1];
      const uint8_t* const x = static_cast<const uint8_t*>(a.x) + static_cast<int64_t>(row) * a.x_row;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int k = wave * 64 + 16 * g; k < ((a.k + 63) & ~63); k += kRowWaves * 64) {
        const bool there = k < a.k;  // (in the last columns lanes may have none)
        const int at = there ? k : 0;
        i32x4 raw = load128(x + at);
        Pack8 xs[2], as[2];
        as[0].raw = load128(A + at);
        as[1].raw = load128(A + at + 8);
        if (!there) raw = as[0].raw = as[1].raw = i32x4{0, 0, 0, 0};
        widen<T>(raw, xs);
        acc = Mma<T>::run(as[0], xs[0], acc);
        acc = Mma<T>::run(as[1], xs[1], acc);
      }
      f32x4 settled[1] = {acc};
      mfma_settle(settled);
      parts[wave][lane] = settled[0];
      __syncthreads();
      if (wave == 0 && i0 + m < count) {
        f32x4 sum = parts[0][lane];
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) sum += parts[w][lane];
        store_h(a, row, slice, first + 4 * g, sum);
      }
      __syncthreads();
    }
  }
}

// The rows by slot, those without one last: a counting sort by one workgroup.  Where in its slot a row comes is left to chance; no result depends on it.
// Bound by latency: 9392 rows 9 us, 8192 rows of 128 slots 10.8.  (Sixteen workgroups that count all rows and place a share each, or places written side by side from LDS: the same.)
constexpr int kOrderThreads = 1024;
__global__ __launch_bounds__(kOrderThreads) void order_kernel(MloraProjectArgs a) {
  __shared__ int next[MLORA_MAX_SLOTS];
  __shared__ int starts[MLORA_MAX_SLOTS], counts[MLORA_MAX_SLOTS], first_group[MLORA_MAX_SLOTS];
  __shared__ int sums[kOrderThreads / 64], group_sums[kOrderThreads / 64], without;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  static_assert(MLORA_MAX_SLOTS == kOrderThreads, "a slot a thread");
  int32_t* const order = static_cast<int32_t*>(a.workspace);
  int32_t *const slots = order + a.num_rows, *const ends = slots + a.num_rows;
  next[tid] = 0;
  if (tid == 0) {
    without = 0;
    *any_h_beyond(a) = 0;
  }
  __syncthreads();
  // one addition for a wavefront whose rows are of one slot
  auto take = [&](int s, int t) -> int {
    int* const counter = s >= 0 ? next + s : &without;
    const int first = __builtin_amdgcn_readfirstlane(s);
    const unsigned long long live = __ballot(t < a.num_rows);
    if (__ballot(t < a.num_rows && s == first) == live) {
      int at = 0;
      if (lane == 0) at = atomicAdd(counter, __builtin_popcountll(live));
      return __builtin_amdgcn_readfirstlane(at) + __builtin_popcountll(live & ((1ull << lane) - 1));
    }
    return t < a.num_rows ? atomicAdd(counter, 1) : 0;
  };
  // (sixteen rounds' slots are asked for at once: one trip to memory for up to 16384 rows)
  constexpr int kAtOnce = 16;
  int held[kAtOnce];
  auto look_up = [&](int base) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int t = base + i * kOrderThreads + tid;
      held[i] = base + i * kOrderThreads < a.num_rows ? a.token_to_slot[t < a.num_rows ? t : a.num_rows - 1] : -1;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (base + i * kOrderThreads + tid >= a.num_rows || held[i] < 0 || held[i] >= a.num_slots) held[i] = -1;
  };
  const bool few = a.num_rows <= kAtOnce * kOrderThreads;  // (then the first pass's places in the slots are the second's)
  int place[kAtOnce];
  for (int base = 0; base < a.num_rows; base += kAtOnce * kOrderThreads) {
    look_up(base);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) place[i] = base + i * kOrderThreads < a.num_rows ? take(held[i], base + i * kOrderThreads + tid) : 0;
  }
  __syncthreads();
  // exclusive sums over the slots, of their rows and of the groups of up to 64 of them
  const int mine = next[tid], groups = (mine + kGroup - 1) / kGroup;
  int sum = mine, group_sum = groups;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int other = __shfl_up(sum, o, kWave), group_other = __shfl_up(group_sum, o, kWave);
    if (lane >= o) {
      sum += other;
      group_sum += group_other;
    }
  }
  if (lane == 63) {
    sums[wave] = sum;
    group_sums[wave] = group_sum;
  }
  __syncthreads();
  int before = 0, all = 0, groups_before = 0, all_groups = 0;
#pragma unroll
  for (int w = 0; w < kOrderThreads / 64; ++w) {
    before += w < wave ? sums[w] : 0;
    groups_before += w < wave ? group_sums[w] : 0;
    all += sums[w];
    all_groups += group_sums[w];
  }
  const int start = before + sum - mine;
  starts[tid] = start;
  counts[tid] = mine;
  first_group[tid] = groups_before + group_sum - groups;
  next[tid] = start;
  if (tid == 0) without = all;
  __syncthreads();
  for (int base = 0; base < a.num_rows; base += kAtOnce * kOrderThreads) {
    if (!few) look_up(base);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int t = base + i * kOrderThreads + tid;
      if (base + i * kOrderThreads >= a.num_rows) continue;
      const int at = few ? place[i] + (held[i] >= 0 ? starts[held[i]] : all) : take(held[i], t);
      if (t < a.num_rows) {
        order[at] = t;
        slots[at] = held[i];
        ends[at] = held[i] >= 0 ? starts[held[i]] + counts[held[i]] : a.num_rows;
      }
    }
  }
  // the groups: a slot, its first row in the order, how many; the end is a group of none
  i32x4* const list = group_list(a);
  const int capacity = group_capacity(a.num_rows, a.num_slots);
  for (int e = tid; e < capacity; e += kOrderThreads) {
    int lo = 0, hi = MLORA_MAX_SLOTS;  // first_group[lo] <= e, the last such slot that has rows
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_group[mid] <= e) lo = mid;
      else hi = mid;
    }
    const int in = (e - first_group[lo]) * kGroup;
    list[e] = e < all_groups ? i32x4{lo, starts[lo] + in, counts[lo] - in < kGroup ? counts[lo] - in : kGroup, 0} : i32x4{0, 0, 0, 0};
  }
}

// A group of up to 64 rows of a slot; 16 RB ranks of one slice.  TEAMS of four wavefronts take 128 columns of K each in turn, a wavefront sixteen of the rows.  The columns of the rows and of
// the slot's A come by direct loads into one of a team's two buffers, in whole lines, the 16-byte pieces of a row exchanged so that what the lanes read at once lies in all banks.
// (9392 rows, K = 1024, 2 slices of rank 64 10 us; 8192 rows of 128 slots, K = 4096, 23 us: 100 MB of A, 4.3 TB/s.  The whole call with one team in place of two: 181 and 181 us, 90.7 and 89.0.)
// Four teams, of 32 ranks at most, where that gives a compute unit one workgroup at most: the whole call with two teams and with four, 600 rows of 32 slots of rank 64: k 8192, n 1024 73.9 and 63.9 us, k 1024, n 1536
// 28.3 and 26.8; 2000 rows of 8 slots of rank 32, k 4096, n 4096 66.4 and 64.0.
template <typename T, int RB, int TEAMS> __global__ __launch_bounds__(TEAMS * 256) void shrink8_tiles_kernel(MloraProjectArgs a) {
  constexpr int kStage = kGroup * 128 + 16 * RB * 256;
  extern __shared__ char lds[];
  const int everyone = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), team = everyone >> 2, wave = everyone & 3;
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int ranges = (a.r + 16 * RB - 1) / (16 * RB), slice = blockIdx.y / ranges, first = (blockIdx.y - slice * ranges) * 16 * RB;
  const int32_t* const order = static_cast<const int32_t*>(a.workspace);
  const i32x4 group = group_list(a)[blockIdx.x];
  const int slot = __builtin_amdgcn_readfirstlane(group[0]), t0 = __builtin_amdgcn_readfirstlane(group[1]), rows = __builtin_amdgcn_readfirstlane(group[2]);
  if (rows == 0) return;
  uint32_t x_off[2], a_off[RB];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = (wave * 2 + i) * 8 + (lane >> 3);
    x_off[i] = static_cast<uint32_t>(order[t0 + (row < rows ? row : rows - 1)]) * static_cast<uint32_t>(a.x_row) + 16 * ((lane & 7) ^ (((lane >> 4) & 3) + 4 * i));
  }
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const int at = (wave * RB + i) * 4 + (lane >> 4), j = first + at;
    a_off[i] = static_cast<uint32_t>(j < a.r ? j : a.r - 1) * static_cast<uint32_t>(a.k) * 2 + 16 * ((lane & 15) ^ (at & 15));
  }
  char* const mine = lds + team * 2 * kStage;
  const uint32_t home = lds_address(mine);
  const int steps = (a.k + 127) / 128, turns = (steps + TEAMS - 1) / TEAMS;
  const char* const x_base = static_cast<const char*>(a.x);
  const char* const a_base = static_cast<const char*>(a.slices[slice].a) + static_cast<int64_t>(slot) * a.r * a.k * 2;
  auto request = [&](int turn) {
    const int k0 = (turn * TEAMS + team) * 128;
    if (k0 >= a.k) return;
    const uint32_t to = home + (turn & 1) * kStage;
    const bool whole = k0 + 128 <= a.k;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t k = k0;  // (lanes behind the end of a row load its first bytes, which are multiplied by zero)
      if (!whole && k0 + 16 * ((lane & 7) ^ (((lane >> 4) & 3) + 4 * i)) >= a.k) k = 0u - 16 * ((lane & 7) ^ (((lane >> 4) & 3) + 4 * i));
      dma16_from(x_base, x_off[i] + k, to + (wave * 2 + i) * 1024);
    }
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int piece = (lane & 15) ^ (((wave * RB + i) * 4 + (lane >> 4)) & 15);
      uint32_t k = k0 * 2;
      if (!whole && k0 + 8 * piece >= a.k) k = 0u - 16 * piece;
      dma16_from(a_base, a_off[i] + k, to + kGroup * 128 + (wave * RB + i) * 1024);
    }
  };
  f32x4 acc[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) acc[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const bool some = wave * 16 < rows;
  const char* const x_at = mine + (wave * 16 + m) * 128;
  const char* const a_at = mine + kGroup * 128 + m * 256;
  request(0);
  for (int turn = 0; turn < turns; ++turn) {
    wait_lds();
    wait_loads<0>();
    stage_barrier();
    if (turn + 1 < turns) request(turn + 1);
    const int k0 = (turn * TEAMS + team) * 128, stage = (turn & 1) * kStage;
    if (!some || k0 >= a.k) continue;
    Pack8 as[RB][2][2];
    i32x4 raw[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      raw[p] = load128(x_at + stage + 16 * ((4 * p + g) ^ (m >> 1)));
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int v = 0; v < 2; ++v) as[b][p][v].raw = load128(a_at + stage + b * 4096 + 16 * ((8 * p + 2 * g + v) ^ m));
    }
    if (k0 + 128 > a.k) {  // what lies behind the end of a row: zero on both sides
#pragma unroll
      for (int p = 0; p < 2; ++p)
        if (k0 + 64 * p + 16 * g >= a.k) {
          raw[p] = i32x4{0, 0, 0, 0};
#pragma unroll
          for (int b = 0; b < RB; ++b) as[b][p][0].raw = as[b][p][1].raw = i32x4{0, 0, 0, 0};
        }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      Pack8 xs[2];
      widen<T>(raw[p], xs);
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = Mma<T>::run(as[b][p][v], xs[v], acc[b]);
    }
    mfma_settle(acc);
  }
  // the teams' sums meet in the buffers, which nobody reads any more
  wait_lds();
  stage_barrier();
  f32x4* const parts = reinterpret_cast<f32x4*>(lds) + wave * (RB * 64) + lane;
  constexpr int kTeam = 4 * RB * 64;
  if (team) {
#pragma unroll
    for (int b = 0; b < RB; ++b) parts[(team - 1) * kTeam + b * 64] = acc[b];
  }
  __syncthreads();
  if (team == 0 && wave * 16 + m < rows) {
#pragma unroll
    for (int b = 0; b < RB; ++b) {
#pragma unroll
      for (int v = 0; v < TEAMS - 1; ++v) acc[b] += parts[v * kTeam + b * 64];
      if (store_h(a, t0 + wave * 16 + m, slice, first + 16 * b + 4 * g, acc[b])) *any_h_beyond(a) = 1;  // (whoever finds one writes the same)
    }
  }
}

template <typename T, int RB, int TEAMS> void launch_tiles(const MloraProjectArgs* a) {
  constexpr int bytes = TEAMS * 2 * (kGroup * 128 + 16 * RB * 256);
  static_assert(bytes <= kMostLds && (TEAMS - 1) * 4 * RB * 1024 <= bytes, "buffers");
  allow_lds<shrink8_tiles_kernel<T, RB, TEAMS>>(bytes);
  const dim3 grid(static_cast<unsigned>(group_capacity(a->num_rows, a->num_slots)), static_cast<unsigned>(a->num_slices * ((a->r + 16 * RB - 1) / (16 * RB))));
  shrink8_tiles_kernel<T, RB, TEAMS><<<grid, TEAMS * 256, bytes, static_cast<hipStream_t>(a->stream)>>>(*a);
}

template <typename T> void launch(const MloraProjectArgs* a, bool ordered) {
  const hipStream_t stream = static_cast<hipStream_t>(a->stream);
  if (!ordered) {
    const int groups = a->num_slices * ((a->r + 15) / 16), spare = 256 / (a->num_slots * groups), blocks = (a->num_rows + 15) / 16;
    const dim3 grid(static_cast<unsigned>(a->num_slots), static_cast<unsigned>(groups), static_cast<unsigned>(spare < 1 ? 1 : spare < blocks ? spare : blocks));
    shrink8_rows_kernel<T><<<grid, kRowWaves * 64, 0, stream>>>(*a);
    return;
  }
  order_kernel<<<1, kOrderThreads, 0, stream>>>(*a);
  const int64_t groups = static_cast<int64_t>(group_capacity(a->num_rows, a->num_slots)) * a->num_slices;
  const bool few = groups * ((a->r + 31) / 32) <= 256;
  if (a->r <= 16) few ? launch_tiles<T, 1, 4>(a) : launch_tiles<T, 1, 2>(a);
  else if (few) launch_tiles<T, 2, 4>(a);
  else if (a->r <= 32) launch_tiles<T, 2, 2>(a);
  else launch_tiles<T, 4, 2>(a);
}

}  // namespace

int launch_shrink8(const MloraProjectArgs* a, bool ordered) {
  if (a->dtype == MLORA_DTYPE_BF16) launch<__bf16>(a, ordered);
  else launch<_Float16>(a, ordered);
  return check_launch("shrink8");
}

}  // namespace mlora
