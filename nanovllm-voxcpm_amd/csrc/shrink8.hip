// First product of the adapters beside an 8-bit linear: h[t, j] = sum_k x8[t, k] A[slot of t, j, k], for every slice (mlora_project's first launch; the row's scale
// comes with the base product's).
//
// The e4m3 numbers of x become 16-bit ones, exactly, in registers; the wavefronts of a workgroup take 64 columns of K each in turn and add up through LDS.  In front of the
// tiles' linear the rows are put in the order of their slots first, and a workgroup has 64 rows of that order, one slice, up to 64 ranks; few rows stay where they
// are, and a workgroup has the rows of one slot, which it looks for itself, one slice and 16 ranks.
#include "common.h"
#include "launch.h"
#include "project.h"

namespace mlora {

namespace {

// Sixteen e4m3 numbers as two operands of eight.
template <typename T> __device__ __forceinline__ void widen(const i32x4& in, Pack8 (&out)[2]);
template <> __device__ __forceinline__ void widen<__bf16>(const i32x4& in, Pack8 (&out)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i / 2].u[2 * (i % 2)] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[i], 1.0f, false));
    out[i / 2].u[2 * (i % 2) + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[i], 1.0f, true));
  }
}
template <> __device__ __forceinline__ void widen<_Float16>(const i32x4& in, Pack8 (&out)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i / 2].u[2 * (i % 2)] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(in[i], 1.0f, false));
    out[i / 2].u[2 * (i % 2) + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(in[i], 1.0f, true));
  }
}

// h of four ranks from j on of one row, as hi and lo; ranks from r to `ranks` are zero.
__device__ __forceinline__ void store_h(const MloraProjectArgs& a, int row, int slice, int j, const f32x4& sum) {
  const int ranks = padded_ranks(a.r), width = a.num_slices * ranks;
  if (j >= ranks) return;
  __bf16 h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(j + i < a.r ? sum[i] : 0.0f, &h[i], &l[i]);
  uint16_t* const hi = intermediate(a) + static_cast<int64_t>(row) * width + slice * ranks + j;
  __builtin_memcpy(hi, h, 8);
  __builtin_memcpy(hi + static_cast<int64_t>(a.num_rows) * width, l, 8);
}

constexpr int kRowWaves = 8, kRowBatch = kRowWaves * 64;

// The rows of slot blockIdx.x, sixteen of its ranks in one slice.
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
    for (int i0 = 0; i0 < count; i0 += 16) {
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
constexpr int kOrderThreads = 1024;
__global__ __launch_bounds__(kOrderThreads) void order_kernel(MloraProjectArgs a) {
  __shared__ int next[MLORA_MAX_SLOTS];
  __shared__ int sums[kOrderThreads / 64], without;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  static_assert(MLORA_MAX_SLOTS == kOrderThreads, "a slot a thread");
  int32_t* const order = static_cast<int32_t*>(a.workspace);
  int32_t* const slots = order + a.num_rows;
  next[tid] = 0;
  if (tid == 0) without = 0;
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
  const int rounds = (a.num_rows + kOrderThreads - 1) / kOrderThreads;
  for (int i = 0; i < rounds; ++i) {
    const int t = i * kOrderThreads + tid;
    take(slot_of(a, t), t);
  }
  __syncthreads();
  // exclusive sums over the slots
  const int mine = next[tid];
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int other = __shfl_up(sum, o, kWave);
    if (lane >= o) sum += other;
  }
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kOrderThreads / 64; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  next[tid] = before + sum - mine;
  if (tid == 0) without = all;
  __syncthreads();
  for (int i = 0; i < rounds; ++i) {
    const int t = i * kOrderThreads + tid, s = slot_of(a, t);
    const int at = take(s, t);
    if (t < a.num_rows) {
      order[at] = t;
      slots[at] = s;
    }
  }
}

constexpr int kTileWaves = 4, kTileBlocks = 4;  // 64 rows

template <typename T, int RB> __global__ __launch_bounds__(kTileWaves * 64) void shrink8_tiles_kernel(MloraProjectArgs a) {
  constexpr int kBlocks = kTileBlocks;
  __shared__ f32x4 parts[kTileWaves][RB * kBlocks][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int groups = (a.r + 16 * RB - 1) / (16 * RB), slice = blockIdx.y / groups, first = (blockIdx.y - slice * groups) * 16 * RB;
  const int32_t* const order = static_cast<const int32_t*>(a.workspace);
  int mine[kBlocks];
  unsigned left[kBlocks];
  const uint8_t* x[kBlocks];
#pragma unroll
  for (int f = 0; f < kBlocks; ++f) {
    const int at = blockIdx.x * (16 * kBlocks) + 16 * f + m, within = at < a.num_rows ? at : a.num_rows - 1;
    mine[f] = at < a.num_rows ? order[a.num_rows + within] : -1;
    left[f] = static_cast<unsigned>(__ballot(mine[f] >= 0)) & 0xffffu;
    x[f] = static_cast<const uint8_t*>(a.x) + static_cast<int64_t>(order[within]) * a.x_row;
  }
  for (unsigned d = 0;; ++d) {
    int slot = -1;
#pragma unroll
    for (int f = 0; f < kBlocks; ++f)
      if (slot < 0 && left[f]) slot = __builtin_amdgcn_readlane(mine[f], __builtin_ctz(left[f]));
    if (slot < 0) break;
    unsigned has[kBlocks];
#pragma unroll
    for (int f = 0; f < kBlocks; ++f) {
      has[f] = static_cast<unsigned>(__ballot(mine[f] == slot)) & 0xffffu;
      left[f] &= ~has[f];
    }
    if (d % gridDim.z != blockIdx.z) continue;
    const T* const A = static_cast<const T*>(a.slices[slice].a) + static_cast<int64_t>(slot) * a.r * a.k;
    const T* ranks[RB];
    f32x4 acc[RB][kBlocks];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int j = first + 16 * b + m;
      ranks[b] = A + static_cast<int64_t>(j < a.r ? j : a.r - 1) * a.k;
#pragma unroll
      for (int f = 0; f < kBlocks; ++f) acc[b][f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int k = wave * 64 + 16 * g; k < ((a.k + 63) & ~63); k += kTileWaves * 64) {
      const bool there = k < a.k;  // (in the last columns lanes may have none)
      const int at = there ? k : 0;
      Pack8 as[RB][2];
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          as[b][p].raw = load128(ranks[b] + at + 8 * p);
          if (!there) as[b][p].raw = i32x4{0, 0, 0, 0};
        }
#pragma unroll
      for (int f = 0; f < kBlocks; ++f) {
        if (!has[f]) continue;
        i32x4 raw = load128(x[f] + at);
        if (!there) raw = i32x4{0, 0, 0, 0};
        Pack8 xs[2];
        widen<T>(raw, xs);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          acc[b][f] = Mma<T>::run(as[b][0], xs[0], acc[b][f]);
          acc[b][f] = Mma<T>::run(as[b][1], xs[1], acc[b][f]);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      mfma_settle(acc[b]);
#pragma unroll
      for (int f = 0; f < kBlocks; ++f) parts[wave][b * kBlocks + f][lane] = acc[b][f];
    }
    __syncthreads();
    // a wavefront adds up every fourth block of rows
#pragma unroll
    for (int f = 0; f < kBlocks; ++f) {
      if (f % kTileWaves != wave) continue;
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        f32x4 sum = parts[0][b * kBlocks + f][lane];
#pragma unroll
        for (int w = 1; w < kTileWaves; ++w) sum += parts[w][b * kBlocks + f][lane];
        if (mine[f] == slot) store_h(a, blockIdx.x * (16 * kBlocks) + 16 * f + m, slice, first + 16 * b + 4 * g, sum);
      }
    }
    __syncthreads();
  }
}

template <typename T> void launch(const MloraProjectArgs* a, bool ordered) {
  const hipStream_t stream = static_cast<hipStream_t>(a->stream);
  if (!ordered) {
    const dim3 grid(static_cast<unsigned>(a->num_slots), static_cast<unsigned>(a->num_slices * ((a->r + 15) / 16)));
    shrink8_rows_kernel<T><<<grid, kRowWaves * 64, 0, stream>>>(*a);
    return;
  }
  order_kernel<<<1, kOrderThreads, 0, stream>>>(*a);
  const unsigned tiles = static_cast<unsigned>((a->num_rows + 16 * kTileBlocks - 1) / (16 * kTileBlocks));
  const int blocks = a->r <= 16 ? 1 : a->r <= 32 ? 2 : 4;
  const unsigned columns = static_cast<unsigned>(a->num_slices * ((a->r + 16 * blocks - 1) / (16 * blocks)));
  unsigned together = 1024 / (tiles * columns);  // different slots of a tile side by side, as long as that is about what fills the chip
  together = together < 1 ? 1 : together > 16 ? 16 : together;
  const dim3 grid(tiles, columns, together);
  if (blocks == 1) shrink8_tiles_kernel<T, 1><<<grid, kTileWaves * 64, 0, stream>>>(*a);
  else if (blocks == 2) shrink8_tiles_kernel<T, 2><<<grid, kTileWaves * 64, 0, stream>>>(*a);
  else shrink8_tiles_kernel<T, 4><<<grid, kTileWaves * 64, 0, stream>>>(*a);
}

}  // namespace

int launch_shrink8(const MloraProjectArgs* a, bool ordered) {
  if (a->dtype == MLORA_DTYPE_BF16) launch<__bf16>(a, ordered);
  else launch<_Float16>(a, ordered);
  return check_launch("shrink8");
}

}  // namespace mlora
