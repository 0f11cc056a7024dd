// First product of the adapters beside an 8-bit linear: h[t, j] = xs[t] sum_k x8[t, k] A[slot of t, j, k], for every slice (mlora_project's first launch).
//
// A workgroup has sixteen rows, one slice and up to 64 ranks; its four wavefronts take every fourth 64 columns of K and add up through LDS.  Sixteen rows of x
// meet every different slot among them (their e4m3 numbers become 16-bit ones, exactly, in registers), and a slot's result goes to the rows that have it.
#include "common.h"
#include "launch.h"
#include "project.h"

namespace mlora {

namespace {

constexpr int kWaves = 4;

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

template <typename T, int RB> __global__ __launch_bounds__(kWaves * 64) void shrink8_kernel(MloraProjectArgs a) {
  __shared__ f32x4 parts[kWaves][RB][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int groups = (a.r + 16 * RB - 1) / (16 * RB), slice = blockIdx.y / groups, first_rank = (blockIdx.y - slice * groups) * 16 * RB;
  const int row = blockIdx.x * 16 + m, mine = slot_of(a, row);
  int list;
  const int count = different(mine, lane, &list);
  const uint8_t* x = static_cast<const uint8_t*>(a.x) + static_cast<int64_t>(row < a.num_rows ? row : a.num_rows - 1) * a.x_row;
  const int ranks = padded_ranks(a.r), width = a.num_slices * ranks;
  uint16_t* hi = static_cast<uint16_t*>(a.workspace);
  uint16_t* lo = hi + static_cast<int64_t>(a.num_rows) * width;
  for (int d = blockIdx.z; d < count; d += gridDim.z) {
    const int slot = __builtin_amdgcn_readlane(list, d);
    const T* A = static_cast<const T*>(a.slices[slice].a) + static_cast<int64_t>(slot) * a.r * a.k;
    const T* rows[RB];
    f32x4 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int j = first_rank + 16 * b + m;
      rows[b] = A + static_cast<int64_t>(j < a.r ? j : a.r - 1) * a.k;
      acc[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int k = wave * 64 + 16 * g; k < ((a.k + 63) & ~63); k += kWaves * 64) {
      const bool there = k < a.k;  // (in the last columns lanes may have none)
      const int at = there ? k : 0;
      i32x4 raw = load128(x + at);
      if (!there) raw = i32x4{0, 0, 0, 0};
      Pack8 xs[2], as[2];
      widen<T>(raw, xs);
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        as[0].raw = load128(rows[b] + at);
        as[1].raw = load128(rows[b] + at + 8);
        if (!there) as[0].raw = as[1].raw = i32x4{0, 0, 0, 0};
        acc[b] = Mma<T>::run(as[0], xs[0], acc[b]);
        acc[b] = Mma<T>::run(as[1], xs[1], acc[b]);
      }
    }
    mfma_settle(acc);
#pragma unroll
    for (int b = 0; b < RB; ++b) parts[wave][b][lane] = acc[b];
    __syncthreads();
    for (int b = wave; b < RB; b += kWaves) {
      f32x4 sum = parts[0][b][lane];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += parts[w][b][lane];
      const int j = first_rank + 16 * b + 4 * g;
      if (mine == slot && j < ranks) {
        const float scale = a.x_scales[row];
        __bf16 h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split(j + i < a.r ? sum[i] * scale : 0.0f, &h[i], &l[i]);
        const int64_t at = static_cast<int64_t>(row) * width + slice * ranks + j;
        __builtin_memcpy(hi + at, h, 8);
        __builtin_memcpy(lo + at, l, 8);
      }
    }
    __syncthreads();
  }
}

template <typename T> void launch(const MloraProjectArgs* a) {
  const hipStream_t stream = static_cast<hipStream_t>(a->stream);
  const unsigned tiles = static_cast<unsigned>((a->num_rows + 15) / 16);
  const int blocks = a->r <= 16 ? 1 : a->r <= 32 ? 2 : 4;
  const unsigned columns = static_cast<unsigned>(a->num_slices * ((a->r + 16 * blocks - 1) / (16 * blocks)));
  unsigned together = 1024 / (tiles * columns);  // different slots of a tile side by side, as long as that is about what fills the chip
  together = together < 1 ? 1 : together > 16 ? 16 : together;
  const dim3 grid(tiles, columns, together);
  if (blocks == 1) shrink8_kernel<T, 1><<<grid, kWaves * 64, 0, stream>>>(*a);
  else if (blocks == 2) shrink8_kernel<T, 2><<<grid, kWaves * 64, 0, stream>>>(*a);
  else shrink8_kernel<T, 4><<<grid, kWaves * 64, 0, stream>>>(*a);
}

}  // namespace

int launch_shrink8(const MloraProjectArgs* a) {
  if (a->dtype == MLORA_DTYPE_BF16) launch<__bf16>(a);
  else launch<_Float16>(a);
  return check_launch("shrink8");
}

}  // namespace mlora
