// The rows between the linears of a decoder: mlora_add_rms_norm, mlora_silu_mul and mlora_quantize_rows, to the element type or to e4m3 with an fp32 scale a row.
//
// Of a row z (what stands in front of the row's own factor f: the norm's rsqrt(mean(sum^2) + eps), else 1) the 8-bit form is
//   scale = max(max|z f| / 448, 2^-100),   values = e4m3(z f / scale),
// each step rounded as it is written: the 8-bit form of a row is that of its fp32 form, and scale and values belong together.  Everything is fp32; sums of squares are taken element by element in a lane, then over lanes, then over wavefronts.
//
// Bound by memory: a row is read once into registers, reduced and written.  A lane holds pieces of eight elements side by side: of rows whose elements come in eights and that start
// on 16 bytes in one or two loads, of others one by one, to the same sums in the same order: where a row lies does not change what comes out.
// (16 bytes a load is what counts: as unaligned copies, which the compiler splits, the norm of 9392 rows of 1024 bf16 took 20 us and the gate of 9392 rows of 2 x 4096 took 44.)
// Few rows cost a launch and one trip to memory: the lanes meet between registers, and up to 1024 elements are one wavefront's.
// Measured (graph replay): norm with residual of 9392 rows of 1024 bf16 14.0 us (67 MB, 4.8 TB/s; an elementwise sum of two such tensors 10.4 for 58 MB), of 3001 rows of 2048 fp16 10.0 us (49 MB); gate of 9392 rows of 2 x 4096 bf16 31.3 us (6.1 TB/s);
// one row 3.0 us.  Workgroups that stay and fetch their next row ahead gained nothing at any width.
#include "common.h"
#include "launch.h"

// Products and sums round as they are written, in every variant alike.
#pragma clang fp contract(off)

namespace mlora {

namespace {

constexpr float kTop = 448.0f;            // largest e4m3 number
constexpr float kLeastScale = 0x1p-100f;  // a row of zeros has a scale all the same, and 448 / max|z| no overflow

enum Op { kPlain, kNorm, kGate };

// Eight elements side by side, piece c of thread `at`.
template <typename T> struct Piece {
  static constexpr int kWords = sizeof(T) * 8 / 16;
  union {
    i32x4 words[kWords];
    T e[8];
  };
};
template <int THREADS> __device__ __forceinline__ int element(int c, int at, int i) { return (c * THREADS + at) * 8 + i; }

template <typename T, bool VEC, int THREADS> __device__ __forceinline__ void load_piece(const T* row, int width, int c, int at, Piece<T>& to) {
  if constexpr (VEC) {
    if (element<THREADS>(c, at, 0) < width) {
#pragma unroll
      for (int w = 0; w < Piece<T>::kWords; ++w) to.words[w] = load128(row + element<THREADS>(c, at, 0) + w * (16 / sizeof(T)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = element<THREADS>(c, at, i);
      to.e[i] = row[e < width ? e : 0];
    }
  }
}
template <typename T, bool VEC, int THREADS> __device__ __forceinline__ void store_piece(T* row, int width, int c, int at, const float (&in)[8]) {
  Piece<T> out;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v = in[i];
    asm("" : "+v"(v));  // (else a product and its conversion to fp16 are made one, with one rounding, in some variants and not in others)
    out.e[i] = from_f32<T>(v);
  }
  if constexpr (VEC) {
    if (element<THREADS>(c, at, 0) < width) {
#pragma unroll
      for (int w = 0; w < Piece<T>::kWords; ++w) store128(row + element<THREADS>(c, at, 0) + w * (16 / sizeof(T)), out.words[w]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (element<THREADS>(c, at, i) < width) row[element<THREADS>(c, at, i)] = out.e[i];
  }
}
template <bool VEC, int THREADS> __device__ __forceinline__ void store_piece8(uint8_t* row, int width, int c, int at, const float (&in)[8]) {
  u32x2 words;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * i], in[4 * i + 1], 0, false);
    words[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(in[4 * i + 2], in[4 * i + 3], low, true));
  }
  if constexpr (VEC) {
    if (element<THREADS>(c, at, 0) < width) *reinterpret_cast<u32x2*>(row + element<THREADS>(c, at, 0)) = words;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (element<THREADS>(c, at, i) < width) row[element<THREADS>(c, at, i)] = static_cast<uint8_t>(words[i / 4] >> (8 * (i % 4)));
  }
}

// max|z| as bits: among them NaN is the largest, so a row that holds one has no other maximum.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

// What the lane at the other end of a pair holds: neighbours, pairs, groups of four and of eight mirrored, then halves of 32 and of 64 lanes.  (All of it between registers, without LDS.)
template <int STEP> __device__ __forceinline__ uint32_t other_of(uint32_t v) {
  if constexpr (STEP == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (threadIdx.x & 16) ? r[0] : r[1];
  } else if constexpr (STEP == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
  } else {
    constexpr int kControl = STEP == 1 ? 0xb1 : STEP == 2 ? 0x4e : STEP == 4 ? 0x141 : 0x140;
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kControl, 0xf, 0xf, true));
  }
}
template <int STEP> __device__ __forceinline__ void reduce_step(float& sum, uint32_t& top) {
  sum += __uint_as_float(other_of<STEP>(__float_as_uint(sum)));
  top = larger(top, other_of<STEP>(top));
}

// Sum and maximum over the THREADS threads of a row; every thread gets them.
template <int THREADS> __device__ __forceinline__ void reduce(float& sum, uint32_t& top) {
  reduce_step<1>(sum, top);
  reduce_step<2>(sum, top);
  reduce_step<4>(sum, top);
  reduce_step<8>(sum, top);
  reduce_step<16>(sum, top);
  reduce_step<32>(sum, top);
  if constexpr (THREADS > 64) {
    constexpr int kWaves = THREADS / 64;
    __shared__ float sums[kWaves];
    __shared__ uint32_t tops[kWaves];
    const int wave = threadIdx.x >> 6;
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

// What a piece of a row is made of, as it lies in memory: x and the residual, or gate and up.
template <typename T> struct Held {
  Piece<T> x, other;
};
template <typename T, Op OP, bool VEC, int THREADS> __device__ __forceinline__ void load_held(const MloraRowsArgs& a, const RowsOf<T>& r, int c, int at, Held<T>& to) {
  load_piece<T, VEC, THREADS>(r.x, a.width, c, at, to.x);
  if constexpr (OP == kGate) load_piece<T, VEC, THREADS>(r.x + a.width, a.width, c, at, to.other);
  if constexpr (OP == kNorm)
    if (r.residual) load_piece<T, VEC, THREADS>(r.residual, a.width, c, at, to.other);
}
template <typename T, bool VEC, int THREADS> __device__ __forceinline__ void load_weight(const MloraRowsArgs& a, int c, int at, float (&w)[8]) {
  if (a.weight32) {
    Piece<float> raw;
    load_piece<float, VEC, THREADS>(static_cast<const float*>(a.weight), a.width, c, at, raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = raw.e[i];
  } else {
    Piece<T> raw;
    load_piece<T, VEC, THREADS>(static_cast<const T*>(a.weight), a.width, c, at, raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = to_f32(raw.e[i]);
  }
}
// z of a piece, and what it adds to the sum of squares and the maximum; the sum in front of the norm is stored.
template <typename T, Op OP, bool VEC, int THREADS>
__device__ __forceinline__ void row_piece(const MloraRowsArgs& a, const RowsOf<T>& r, int c, int at, const Held<T>& held, const float (&w)[8], float (&z)[8], float& squares, uint32_t& top) {
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = to_f32(held.x.e[i]);
  if constexpr (OP == kNorm) {
    if (r.residual) {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = to_f32(from_f32<T>(z[i] + to_f32(held.other.e[i])));
      store_piece<T, VEC, THREADS>(r.sum, a.width, c, at, z);
    }
  } else if constexpr (OP == kGate) {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = z[i] * __builtin_amdgcn_rcpf(1.0f + __expf(-z[i])) * to_f32(held.other.e[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool there = element<THREADS>(c, at, i) < a.width;
    if constexpr (OP == kNorm) {
      const float v = there ? z[i] : 0.0f;
      squares = __builtin_fmaf(v, v, squares);
      z[i] *= w[i];
    }
    top = larger(top, there ? magnitude(z[i]) : 0);
  }
}

// The row's factor and, for 8 bits, its scale, from the whole row's sums; one thread writes the scale.
//
// Quotients z / scale come from the scale's inverse and one correction, q + (z - q scale) / scale, which is the nearest fp32 number (tried for every scale's mantissa and every z whose quotient is within four
// steps of a tie of e4m3, 3e9 quotients): three instructions where a division takes ten (norm of 9392 rows of 1024: 16.5 us by divisions, 14.0 so; gate of 9392 rows of 2 x 4096: 37.9 and 31.3).  Scales so small that
// the rest z - q scale has no bits left, infinities and NaN are divided by.
struct Factor {
  float f, scale, inverse;  // the last: 0 where it is not used
};
template <Op OP, bool OUT8> __device__ __forceinline__ Factor row_factor(const MloraRowsArgs& a, int row, float squares, uint32_t top, bool writes) {
  const float f = OP == kNorm ? rsqrtf(squares / static_cast<float>(a.width) + a.eps) : 1.0f;
  if constexpr (!OUT8) return Factor{f, 1.0f, 0.0f};
  const float exact = __uint_as_float(top) * f / kTop, scale = exact < kLeastScale ? kLeastScale : exact;
  if (writes) a.scales[row] = scale;
  return Factor{f, scale, scale >= 0x1p-60f && scale <= 0x1p120f ? 1.0f / scale : 0.0f};
}
template <typename T, Op OP, bool OUT8, bool VEC, int THREADS> __device__ __forceinline__ void write_piece(const MloraRowsArgs& a, const RowsOf<T>& r, int c, int at, const Factor& factor, float (&z)[8]) {
  if constexpr (OP == kNorm) {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] *= factor.f;
  }
  if constexpr (OUT8) {
    if (factor.inverse != 0.0f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = z[i] * factor.inverse;
        z[i] = __builtin_fmaf(-__builtin_fmaf(q, factor.scale, -z[i]), factor.inverse, q);  // (-0 stays what it is)
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = z[i] / factor.scale;
    }
  }
  if constexpr (OUT8) store_piece8<VEC, THREADS>(r.out8, a.width, c, at, z);
  else store_piece<T, VEC, THREADS>(r.out, a.width, c, at, z);
}

// A row by THREADS threads, PIECES pieces each in registers; workgroups of fewer than 256 threads a row take several rows.
template <typename T, Op OP, bool OUT8, bool VEC, int THREADS, int PIECES> __global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void rows_kernel(MloraRowsArgs a) {
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
  const int row = blockIdx.x * kRows + threadIdx.x / THREADS, at = threadIdx.x % THREADS;
  if (row >= a.num_rows) return;  // (whole wavefronts; rows that share a workgroup do not meet)
  const RowsOf<T> r = rows_of<T>(a, row);
  Held<T> held[PIECES];
  float weight[PIECES][8], z[PIECES][8], squares = 0.0f;
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < PIECES; ++c) load_held<T, OP, VEC, THREADS>(a, r, c, at, held[c]);
  if constexpr (OP == kNorm) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c) load_weight<T, VEC, THREADS>(a, c, at, weight[c]);
  }
#pragma unroll
  for (int c = 0; c < PIECES; ++c) row_piece<T, OP, VEC, THREADS>(a, r, c, at, held[c], weight[c], z[c], squares, top);
  reduce<THREADS>(squares, top);
  const Factor factor = row_factor<OP, OUT8>(a, row, squares, top, at == 0);
#pragma unroll
  for (int c = 0; c < PIECES; ++c) write_piece<T, OP, OUT8, VEC, THREADS>(a, r, c, at, factor, z[c]);
}

// Rows of any width: read twice, the second time the sum where this thread stored it.
template <typename T, Op OP, bool OUT8, bool VEC> __global__ __launch_bounds__(1024) void long_rows_kernel(MloraRowsArgs a) {
  const int row = blockIdx.x, at = threadIdx.x, pieces = (a.width + 8191) / 8192;
  RowsOf<T> r = rows_of<T>(a, row);
  Held<T> held;
  float z[8], weight[8], squares = 0.0f;
  uint32_t top = 0;
  for (int c = 0; c < pieces; ++c) {
    load_held<T, OP, VEC, 1024>(a, r, c, at, held);
    if constexpr (OP == kNorm) load_weight<T, VEC, 1024>(a, c, at, weight);
    row_piece<T, OP, VEC, 1024>(a, r, c, at, held, weight, z, squares, top);
  }
  reduce<1024>(squares, top);
  const Factor factor = row_factor<OP, OUT8>(a, row, squares, top, at == 0);
  if (OP == kNorm && r.residual) {
    r.x = r.sum;
    r.residual = nullptr;
  }
  for (int c = 0; c < pieces; ++c) {
    load_held<T, OP, VEC, 1024>(a, r, c, at, held);
    if constexpr (OP == kNorm) load_weight<T, VEC, 1024>(a, c, at, weight);
    row_piece<T, OP, VEC, 1024>(a, r, c, at, held, weight, z, squares, top);
    write_piece<T, OP, OUT8, VEC, 1024>(a, r, c, at, factor, z);
  }
}

template <typename T, Op OP, bool OUT8, bool VEC, int THREADS, int PIECES> void launch_one(const MloraRowsArgs* a) {
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1, kThreads = THREADS < 256 ? 256 : THREADS;
  rows_kernel<T, OP, OUT8, VEC, THREADS, PIECES><<<static_cast<unsigned>((a->num_rows + kRows - 1) / kRows), kThreads, 0, static_cast<hipStream_t>(a->stream)>>>(*a);
}
template <typename T, Op OP, bool OUT8, bool VEC> int launch_rows(const MloraRowsArgs* a) {
  if (a->width <= 512) launch_one<T, OP, OUT8, VEC, 64, 1>(a);
  else if (a->width <= 1024) launch_one<T, OP, OUT8, VEC, 64, 2>(a);
  else if (a->width <= 2048) launch_one<T, OP, OUT8, VEC, 256, 1>(a);
  else if (a->width <= 4096) launch_one<T, OP, OUT8, VEC, 256, 2>(a);
  else if (a->width <= 8192) launch_one<T, OP, OUT8, VEC, 256, 4>(a);
  else if (a->width <= 16384) launch_one<T, OP, OUT8, VEC, 1024, 2>(a);
  else long_rows_kernel<T, OP, OUT8, VEC><<<static_cast<unsigned>(a->num_rows), 1024, 0, static_cast<hipStream_t>(a->stream)>>>(*a);
  return check_launch("rows");
}

bool whole_words(const MloraRowsArgs* a, int size, bool out8) {
  const uintptr_t rows = reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->residual) | reinterpret_cast<uintptr_t>(a->sum) | reinterpret_cast<uintptr_t>(a->weight);
  const uintptr_t strides = static_cast<uintptr_t>((a->x_row | (a->residual ? a->residual_row | a->sum_row : 0)) * size);
  const uintptr_t out = reinterpret_cast<uintptr_t>(a->out) | static_cast<uintptr_t>(a->out_row * (out8 ? 1 : size));
  return a->width % 8 == 0 && ((rows | strides) & 15) == 0 && (out & (out8 ? 7 : 15)) == 0;
}
template <typename T, Op OP, bool OUT8> int launch_type(const MloraRowsArgs* a) {
  return whole_words(a, sizeof(T), OUT8) ? launch_rows<T, OP, OUT8, true>(a) : launch_rows<T, OP, OUT8, false>(a);
}
template <Op OP, bool OUT8> int launch_rows_of(const MloraRowsArgs* a) {
  if (a->dtype == MLORA_DTYPE_BF16) return launch_type<__bf16, OP, OUT8>(a);
  if (a->dtype == MLORA_DTYPE_F16) return launch_type<_Float16, OP, OUT8>(a);
  return launch_type<float, OP, OUT8>(a);
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
