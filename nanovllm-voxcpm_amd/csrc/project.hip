// The linear over 8-bit rows and weights with the adapters of many requests beside it (mlora_project), and its entry point.
//
//   y[t, n] = xs[t] ws[n] sum_k x8[t, k] w8[n, k] + bias[n] + sum_j h[t, j] B[slot of t, n, j]
//
// The base product runs on the 16x16x128 e4m3 matrix instruction, weights as its rows, so that a lane holds consecutive columns of one row of y.  The adapters' second
// product continues in the same accumulators: its contraction is a list of pieces of eight ranks, those of the different slots among sixteen rows one behind the other, in which a
// row's h is zero outside its own slot's.
#include "common.h"
#include "launch.h"
#include "project.h"

namespace mlora {

namespace {

// Sixteen columns of y, up to 16 TF rows; K by the wavefronts, every WAVES-th 128 columns each.
template <typename T, int TF, int WAVES> __global__ __launch_bounds__(WAVES * 64) void project_rows_kernel(MloraProjectArgs a) {
  __shared__ f32x4 parts[WAVES][TF][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, t0 = blockIdx.y * (16 * TF);
  const uint8_t* w = static_cast<const uint8_t*>(a.w) + static_cast<int64_t>(n0 + m < a.n ? n0 + m : a.n - 1) * a.w_row;
  const uint8_t* x[TF];
  f32x4 acc[TF];
#pragma unroll
  for (int f = 0; f < TF; ++f) {
    const int t = t0 + 16 * f + m;
    x[f] = static_cast<const uint8_t*>(a.x) + static_cast<int64_t>(t < a.num_rows ? t : a.num_rows - 1) * a.x_row;
    acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int base = wave * 128; base < a.k; base += WAVES * 128) {
    Eight ws, xs[TF];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int k = base + 64 * p + 16 * g;
      const bool there = k < a.k;  // (else zeros of x, and some of w's row, which is NaN only where y is)
      ws.piece[p] = load128(w + (there ? k : 0));
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        xs[f].piece[p] = load128(x[f] + (there ? k : 0));
        if (!there) xs[f].piece[p] = i32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int f = 0; f < TF; ++f) acc[f] = mma8(ws, xs[f], acc[f]);
  }
  mfma_settle(acc);
  float scales[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) scales[i] = n0 + 4 * g + i < a.n ? a.w_scales[n0 + 4 * g + i] : 0.0f;
  const int ranks = padded_ranks(a.r), pieces = ranks / 8, width = a.num_slices * ranks;
  const uint16_t* hi = intermediate(a);
  const uint16_t* lo = hi + static_cast<int64_t>(a.num_rows) * width;
  const bool words = a.r % 8 == 0;
#pragma unroll
  for (int f = 0; f < TF; ++f) {
    const int t = t0 + 16 * f + m;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[f][i] *= scales[i];
    if (!a.num_slices) continue;
    const int mine = slot_of(a, t);
    int list;
    const int count = different(mine, lane, &list);
    for (int s = 0; s < a.num_slices; ++s) {
      const int columns = a.slices[s].n, n = n0 + m - a.slices[s].y_col;
      if (n0 + 16 <= a.slices[s].y_col || n0 >= a.slices[s].y_col + columns) continue;
      for (int c0 = 4 * wave; c0 < count * pieces; c0 += 4 * WAVES) {
        const int c = c0 + g, d = c / pieces < count ? c / pieces : count - 1, first = 8 * (c - c / pieces * pieces);
        const int slot = __shfl(list, d, kWave);
        const bool there = c < count * pieces;
        Pack8 raw, h[2];
        raw.raw = h[0].raw = h[1].raw = i32x4{0, 0, 0, 0};
        if (there && n >= 0 && n < columns) {
          const T* b = static_cast<const T*>(a.slices[s].b) + (static_cast<int64_t>(slot) * columns + n) * a.r + first;
          if (words) {
            raw.raw = load128(b);
          } else {
            T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (first + i < a.r) e[i] = b[i];
          }
        }
        if (there && mine == slot) {
          const int64_t at = static_cast<int64_t>(t) * width + s * ranks + first;
          h[0].raw = load128(hi + at);
          if constexpr (kParts<T> == 2) h[1].raw = load128(lo + at);
        }
        if (__ballot(any_beyond<T>(raw))) {  // (the four pieces of the list one behind the other)
          for (int v = 0; v < 4 && c0 + v < count * pieces; ++v) {
            const int of = (c0 + v) / pieces, slot = __builtin_amdgcn_readlane(list, of);
            const int64_t at = static_cast<int64_t>(t) * width + s * ranks;
            if (mine == slot)
              add_slowly(static_cast<const T*>(a.slices[s].b) + static_cast<int64_t>(slot) * columns * a.r, columns, n0 + 4 * g - a.slices[s].y_col, a.r, 8 * (c0 + v - of * pieces), 8,
                         hi + at, kParts<T> == 2 ? lo + at : nullptr, acc[f]);
          }
          continue;
        }
        BPiece<T> b;
        b.from(raw);
        acc[f] = Mma<__bf16>::run(b.hi, h[0], acc[f]);
        if constexpr (kParts<T> == 2) {
          acc[f] = Mma<__bf16>::run(b.hi, h[1], acc[f]);
          acc[f] = Mma<__bf16>::run(b.lo, h[0], acc[f]);
        }
      }
    }
  }
  mfma_settle(acc);
#pragma unroll
  for (int f = 0; f < TF; ++f) parts[wave][f][lane] = acc[f];
  __syncthreads();
  for (int f = wave; f < TF; f += WAVES) {
    const int t = t0 + 16 * f + m, n = n0 + 4 * g;
    if (t >= a.num_rows) continue;
    f32x4 sum = parts[0][f][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) sum += parts[v][f][lane];
    const float scale = a.x_scales[t];
    T* y = static_cast<T*>(a.y) + static_cast<int64_t>(t) * a.y_row + n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.n) y[i] = from_f32<T>(__builtin_fmaf(sum[i], scale, a.bias ? to_f32(static_cast<const T*>(a.bias)[n + i]) : 0.0f));
  }
}

template <typename T> void launch(const MloraProjectArgs* a) {
  const hipStream_t stream = static_cast<hipStream_t>(a->stream);
  const unsigned columns = static_cast<unsigned>((a->n + 15) / 16);
  auto rows = [&](int tile) { return dim3(columns, static_cast<unsigned>((a->num_rows + tile - 1) / tile)); };
  if (a->num_rows <= 16) project_rows_kernel<T, 1, 8><<<rows(16), 512, 0, stream>>>(*a);
  else if (a->num_rows <= 32) project_rows_kernel<T, 2, 8><<<rows(32), 512, 0, stream>>>(*a);
  else project_rows_kernel<T, 4, 8><<<rows(64), 512, 0, stream>>>(*a);
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

size_t workspace_bytes(const MloraProjectArgs* a) {
  return static_cast<size_t>(order_bytes(a->num_rows, a->num_slots)) + static_cast<size_t>(a->num_rows) * a->num_slices * padded_ranks(a->r) * (a->dtype == MLORA_DTYPE_F16 ? 4 : 2);
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

int project_kind(const MloraProjectArgs* a) {
  const int forced = env_int("MLORA_TILE8", 0);
  if (forced) return forced - 1;
  if (a->num_rows <= 256 || !tiles8_supported(a)) return kRows;
  return a->num_rows > 2048 ? kTiles128 : kTiles64;
}

int launch_project_rows(const MloraProjectArgs* a) {
  if (a->dtype == MLORA_DTYPE_BF16) launch<__bf16>(a);
  else launch<_Float16>(a);
  return check_launch("project");
}

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_project(const MloraProjectArgs* a) {
  const int rc = check_project(a);
  if (rc) return rc == kNothingToDo ? 0 : rc;
  const int kind = project_kind(a);
  if (a->num_slices)
    if (const int failed = launch_shrink8(a, kind != kRows)) return failed;
  return kind == kRows ? launch_project_rows(a) : launch_tiles8(a, kind);
}

extern "C" size_t mlora_project_workspace_bytes(const MloraProjectArgs* a) {
  return a && a->num_rows > 0 && a->n > 0 && a->num_slices > 0 && a->num_slices <= MLORA_MAX_SLICES && a->r > 0 && a->r <= MLORA_MAX_RANK ? workspace_bytes(a) : 0;
}
