// The rows between the linears of a decoder: mlora_add_rms_norm, mlora_silu_mul and mlora_quantize_rows, to the element type or to e4m3 with an fp32 scale a row.
//
// Of a row z (what stands in front of the row's own factor f: the norm's rsqrt(mean(sum^2) + eps), else 1) the 8-bit form is
//   scale = max(f max|z| / 448, 2^-100),   values = e4m3(z f / scale) = e4m3(z 448 / max|z|) where the bound does not hold,
// so the values need no f at all, and of 16-bit inputs and weights z = sum * weight is exact: one rounding for 448 / max|z|, one for its product, then
// the one to 8 bits.  Everything is fp32; sums of squares are taken eight elements a lane, then over lanes, then over wavefronts.
//
// Bound by memory: a row is read once into registers (a wavefront, 256 or 1024 threads a row, up to four pieces of eight elements a thread), reduced and written.
#include "common.h"
#include "launch.h"

namespace mlora {

namespace {

constexpr float kTop = 448.0f;            // largest e4m3 number
constexpr float kLeastScale = 0x1p-100f;  // a row of zeros has a scale all the same, and 448 / max|z| no overflow

enum Op { kPlain, kNorm, kGate };

template <typename T> struct Piece {
  static constexpr int kWords = sizeof(T) * 8 / 16;
  i32x4 raw[kWords];
};
// Eight elements from `p`: whole 16-byte words, which need not be aligned, where `left` allows it, else the ones that are there.
template <typename T> struct __attribute__((packed)) Loose { Piece<T> v; };
template <typename T> __device__ __forceinline__ void load_piece(const T* p, int left, float (&out)[8]) {
  union {
    Piece<T> piece;
    T e[8];
  } u;
  if (left >= 8) {
    __builtin_memcpy(&u, p, sizeof(u));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) u.e[i] = i < left ? p[i] : from_f32<T>(0.0f);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = to_f32(u.e[i]);
}
template <typename T> __device__ __forceinline__ void store_piece(T* p, int left, const float (&in)[8]) {
  union {
    Piece<T> piece;
    T e[8];
  } u;
#pragma unroll
  for (int i = 0; i < 8; ++i) u.e[i] = from_f32<T>(in[i]);
  if (left >= 8) {
    __builtin_memcpy(p, &u, sizeof(u));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = u.e[i];
  }
}
__device__ __forceinline__ void store_piece8(uint8_t* p, int left, const float (&in)[8]) {
  union {
    int w[2];
    uint8_t e[8];
  } u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    u.w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * i], in[4 * i + 1], 0, false);
    u.w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * i + 2], in[4 * i + 3], u.w[i], true);
  }
  if (left >= 8) {
    __builtin_memcpy(p, &u, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = u.e[i];
  }
}

// max|z| as bits: among them NaN is the largest, so a row that holds one has no other maximum.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Sum and maximum over the THREADS threads of a row; every thread gets them.
template <int THREADS> __device__ __forceinline__ void reduce(float& sum, uint32_t& top) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    sum += __shfl_xor(sum, o, kWave);
    top = larger(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, kWave)));
  }
  if constexpr (THREADS > 64) {
    constexpr int kWaves = THREADS / 64;
    __shared__ float sums[kWaves];
    __shared__ uint32_t tops[kWaves];
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // (of a call before this one everybody has read)
    if ((threadIdx.x & 63) == 0) {
      sums[wave] = sum;
      tops[wave] = top;
    }
    __syncthreads();
    sum = 0.0f;
    top = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      sum += sums[w];
      top = larger(top, tops[w]);
    }
  }
}

template <typename T> struct RowsOf {
  const T* x;
  const T* residual;
  T* sum;
  T* out;
  uint8_t* out8;
};
template <typename T> __device__ __forceinline__ RowsOf<T> rows_of(const MloraRowsArgs& a, int row) {
  RowsOf<T> r;
  r.x = static_cast<const T*>(a.x) + row * a.x_row;
  r.residual = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_row : nullptr;
  r.sum = a.residual ? static_cast<T*>(a.sum) + row * a.sum_row : nullptr;
  r.out = static_cast<T*>(a.out) + row * a.out_row;
  r.out8 = static_cast<uint8_t*>(a.out) + row * a.out_row;
  return r;
}

// z of the eight elements from `first` on, and what they add to the sum of squares.  With `again` the sum in front of the norm is read back where this thread stored it.
template <typename T, Op OP> __device__ __forceinline__ float row_piece(const MloraRowsArgs& a, const RowsOf<T>& r, int first, bool again, float (&z)[8]) {
  const int left = a.width - first;
  float squares = 0.0f;
  if constexpr (OP == kNorm) {
    if (again && r.sum) {
      load_piece(r.sum + first, left, z);
    } else {
      load_piece(r.x + first, left, z);
      if (r.residual) {
        float other[8];
        load_piece(r.residual + first, left, other);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = to_f32(from_f32<T>(z[i] + other[i]));
        store_piece(r.sum + first, left, z);
      }
    }
    float w[8];
    if (a.weight32) load_piece(static_cast<const float*>(a.weight) + first, left, w);
    else load_piece(static_cast<const T*>(a.weight) + first, left, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      squares += z[i] * z[i];
      z[i] *= w[i];
    }
  } else {
    load_piece(r.x + first, left, z);
    if constexpr (OP == kGate) {
      float up[8];
      load_piece(r.x + a.width + first, left, up);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = z[i] * __builtin_amdgcn_rcpf(1.0f + __expf(-z[i])) * up[i];
    }
  }
  return squares;
}

// What a z is multiplied with to become the output, from the whole row's sums; lane 0 writes the scale.
template <Op OP, bool OUT8> __device__ __forceinline__ float row_factor(const MloraRowsArgs& a, int row, float squares, uint32_t top, bool writes) {
  const float f = OP == kNorm ? rsqrtf(squares / static_cast<float>(a.width) + a.eps) : 1.0f;
  if constexpr (!OUT8) return f;
  const float most = __uint_as_float(top), exact = most * f / kTop;
  const bool least = exact < kLeastScale;
  if (writes) a.scales[row] = least ? kLeastScale : exact;
  return least ? f / kLeastScale : kTop / most;
}
template <typename T, bool OUT8> __device__ __forceinline__ void write_piece(const RowsOf<T>& r, int first, int left, float factor, float (&z)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] *= factor;
  if constexpr (OUT8) store_piece8(r.out8 + first, left, z);
  else store_piece(r.out + first, left, z);
}

// A row by THREADS threads, PIECES pieces each in registers; workgroups of fewer than 256 threads a row take several rows.
template <typename T, Op OP, bool OUT8, int THREADS, int PIECES>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void rows_kernel(MloraRowsArgs a) {
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
  const int row = blockIdx.x * kRows + threadIdx.x / THREADS, at = threadIdx.x % THREADS;
  if (row >= a.num_rows) return;  // (whole wavefronts; rows that share a workgroup do not meet)
  const RowsOf<T> r = rows_of<T>(a, row);
  float z[PIECES][8], squares = 0.0f;
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < PIECES; ++c) {
    const int first = (c * THREADS + at) * 8;
    if (first < a.width) {
      squares += row_piece<T, OP>(a, r, first, false, z[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = larger(top, magnitude(z[c][i]));
    }
  }
  reduce<THREADS>(squares, top);
  const float factor = row_factor<OP, OUT8>(a, row, squares, top, at == 0);
#pragma unroll
  for (int c = 0; c < PIECES; ++c) {
    const int first = (c * THREADS + at) * 8;
    if (first < a.width) write_piece<T, OUT8>(r, first, a.width - first, factor, z[c]);
  }
}

// Rows of any width: read twice.
template <typename T, Op OP, bool OUT8> __global__ __launch_bounds__(1024) void long_rows_kernel(MloraRowsArgs a) {
  const int row = blockIdx.x;
  const RowsOf<T> r = rows_of<T>(a, row);
  float z[8], squares = 0.0f;
  uint32_t top = 0;
  for (int first = threadIdx.x * 8; first < a.width; first += 8192) {
    squares += row_piece<T, OP>(a, r, first, false, z);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = larger(top, magnitude(z[i]));
  }
  reduce<1024>(squares, top);
  const float factor = row_factor<OP, OUT8>(a, row, squares, top, threadIdx.x == 0);
  for (int first = threadIdx.x * 8; first < a.width; first += 8192) {
    row_piece<T, OP>(a, r, first, true, z);
    write_piece<T, OUT8>(r, first, a.width - first, factor, z);
  }
}

template <typename T, Op OP, bool OUT8> int launch_rows(const MloraRowsArgs* a) {
  const hipStream_t stream = static_cast<hipStream_t>(a->stream);
  const unsigned rows = static_cast<unsigned>(a->num_rows), fours = (rows + 3) / 4;
  if (a->width <= 512) rows_kernel<T, OP, OUT8, 64, 1><<<fours, 256, 0, stream>>>(*a);
  else if (a->width <= 1024) rows_kernel<T, OP, OUT8, 64, 2><<<fours, 256, 0, stream>>>(*a);
  else if (a->width <= 2048) rows_kernel<T, OP, OUT8, 256, 1><<<rows, 256, 0, stream>>>(*a);
  else if (a->width <= 4096) rows_kernel<T, OP, OUT8, 256, 2><<<rows, 256, 0, stream>>>(*a);
  else if (a->width <= 8192) rows_kernel<T, OP, OUT8, 256, 4><<<rows, 256, 0, stream>>>(*a);
  else if (a->width <= 32768) rows_kernel<T, OP, OUT8, 1024, 4><<<rows, 1024, 0, stream>>>(*a);
  else long_rows_kernel<T, OP, OUT8><<<rows, 1024, 0, stream>>>(*a);
  return check_launch("rows");
}

template <Op OP, bool OUT8> int launch_rows_of(const MloraRowsArgs* a) {
  if (a->dtype == MLORA_DTYPE_BF16) return launch_rows<__bf16, OP, OUT8>(a);
  if (a->dtype == MLORA_DTYPE_F16) return launch_rows<_Float16, OP, OUT8>(a);
  return launch_rows<float, OP, OUT8>(a);
}

constexpr int kMostRows = 1 << 24;  // (of 256 threads a row: a launch's dimension has fewer than 2^32 threads)

int check_rows(const MloraRowsArgs* a, const char* what) {
  if (!a) { set_error("%s: NULL args", what); return MLORA_E_INVALID; }
  if (a->num_rows < 0 || a->width < 0) { set_error("%s: negative size", what); return MLORA_E_INVALID; }
  if (a->dtype != MLORA_DTYPE_F32 && a->dtype != MLORA_DTYPE_F16 && a->dtype != MLORA_DTYPE_BF16) {
    set_error("%s: unknown dtype %d", what, a->dtype);
    return MLORA_E_INVALID;
  }
  if (a->num_rows == 0) return kNothingToDo;
  if (a->width == 0) { set_error("%s: rows without elements", what); return MLORA_E_INVALID; }
  if (a->width > INT32_MAX / 4) { set_error("%s: width = %d is more than 2^29", what, a->width); return MLORA_E_TOO_LARGE; }
  if (!a->x || !a->out) { set_error("%s: NULL pointer", what); return MLORA_E_INVALID; }
  const int most = a->width > 8192 ? (1 << 22) - 1 : kMostRows - 1;
  if (a->num_rows > most) { set_error("%s: %d rows of %d elements are more than one launch holds", what, a->num_rows, a->width); return MLORA_E_TOO_LARGE; }
  return 0;
}

}  // namespace

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_add_rms_norm(const MloraRowsArgs* a) {
  const int rc = check_rows(a, "mlora_add_rms_norm");
  if (rc) return rc == kNothingToDo ? 0 : rc;
  if (!a->weight || (a->residual && !a->sum)) { set_error("mlora_add_rms_norm: NULL pointer"); return MLORA_E_INVALID; }
  return a->scales ? launch_rows_of<kNorm, true>(a) : launch_rows_of<kNorm, false>(a);
}

extern "C" int mlora_silu_mul(const MloraRowsArgs* a) {
  const int rc = check_rows(a, "mlora_silu_mul");
  if (rc) return rc == kNothingToDo ? 0 : rc;
  if (a->residual) { set_error("mlora_silu_mul: there is no residual"); return MLORA_E_INVALID; }
  return a->scales ? launch_rows_of<kGate, true>(a) : launch_rows_of<kGate, false>(a);
}

extern "C" int mlora_quantize_rows(const MloraRowsArgs* a) {
  const int rc = check_rows(a, "mlora_quantize_rows");
  if (rc) return rc == kNothingToDo ? 0 : rc;
  if (a->residual || !a->scales) { set_error("mlora_quantize_rows: %s", a->residual ? "there is no residual" : "scales is NULL"); return MLORA_E_INVALID; }
  return launch_rows_of<kPlain, true>(a);
}
