// Norm, rotation and cache store of a batch's query, key and value heads (mlora_rotate_qk); stands where the reference runs its
// rotary embedding and its store_kvcache_kernel (nanovllm_voxcpm/layers/rotary_embedding.py, layers/attention.py:10-50).
//
// A head is W lanes of 16 bytes each (W = dim / 8, in fp32 dim / 4, up to the next power of two): its mean square is a butterfly over
// those lanes, the partner of an element in the other half comes from one of them, in neighbouring pairs from the lane itself.  All of it
// in fp32, one rounding at the end.  Bound by memory: a batch's heads are read once and written once.  A group of W lanes takes a few heads of one token, for
// which it holds the cosines and sines in registers: read anew for every head they would be as many bytes as the head again.
#include "common.h"
#include "launch.h"

namespace mlora {

namespace {

constexpr int kThreads = 256;

template <typename T, bool kAligned> __device__ __forceinline__ void load_chunk(const T* p, float (&x)[16 / sizeof(T)]) {
  constexpr int C = 16 / sizeof(T);
  if constexpr (kAligned) {
    const i32x4 raw = load128(p);
    T e[C];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = to_f32(p[i]);
  }
}

template <typename T, bool kAligned> __device__ __forceinline__ void store_chunk(T* p, const float (&x)[16 / sizeof(T)]) {
  constexpr int C = 16 / sizeof(T);
  T e[C];
#pragma unroll
  for (int i = 0; i < C; ++i) e[i] = from_f32<T>(x[i]);
  if constexpr (kAligned) {
    i32x4 raw;
    __builtin_memcpy(&raw, e, 16);
    store128(p, raw);
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) p[i] = e[i];
  }
}

template <typename T> __device__ __forceinline__ void load_weight(const void* w, bool weights32, int at, float (&out)[16 / sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i)
    out[i] = weights32 ? static_cast<const float*>(w)[at + i] : to_f32(static_cast<const T*>(w)[at + i]);
}

// `width`: lanes of a head; `per`: heads of a group; `chunks`: groups of a token.
template <typename T, bool kAligned>
__global__ __launch_bounds__(kThreads) void rotate_kernel(MloraRotateArgs a, int width, int per, int chunks) {
  constexpr int C = 16 / sizeof(T);
  const int lane = threadIdx.x & 63, c = lane & (width - 1), base = lane - c;
  const long long unit = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) / width;
  const int t = static_cast<int>(unit / chunks), chunk = static_cast<int>(unit - static_cast<long long>(t) * chunks);
  if (t >= a.num_tokens) return;
  const int e0 = c * C;
  const bool mine = e0 < a.dim;
  const int half = a.rotary >> 1;
  const bool turned = e0 < a.rotary;
  const long long position = a.positions64 ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int32_t*>(a.positions)[t];

  // (cos, sin) of this lane's elements: of the pair's number
  float cosine[C], sine[C];
  if (turned) {
    const bool known = position >= 0 && position < a.num_positions;
    const float* row = a.cos_sin + (known ? position : 0) * a.table_row;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int pair = a.interleaved ? (e0 + i) >> 1 : e0 + i < half ? e0 + i : e0 + i - half;
      cosine[i] = known ? row[pair] : __builtin_nanf("");
      sine[i] = known ? row[half + pair] : __builtin_nanf("");
    }
  }
  const int partner = base + (e0 < half ? c + half / C : c - half / C);

  T* stored_k = nullptr;
  T* stored_v = nullptr;
  if (a.slots) {
    const long long slot = a.slots64 ? static_cast<const int64_t*>(a.slots)[t] : static_cast<const int32_t*>(a.slots)[t];
    if (slot >= 0 && slot < static_cast<long long>(a.num_blocks) * a.page) {
      const long long block = slot / a.page, row = slot - block * a.page;
      stored_k = static_cast<T*>(a.k_cache) + block * a.k_block + row * a.k_cache_row;
      stored_v = static_cast<T*>(a.v_cache) + block * a.v_block + row * a.v_cache_row;
    }
  }

  const int all = a.heads + a.kv_heads + (a.v ? a.kv_heads : 0);
  const int first = chunk * per, last = first + per < all ? first + per : all;
  for (int h = first; h < last; ++h) {
    float x[C];
    if (h >= a.heads + a.kv_heads) {  // v: a copy
      const int g = h - a.heads - a.kv_heads;
      if (mine && stored_v) {
        load_chunk<T, kAligned>(static_cast<const T*>(a.v) + t * a.v_row + g * a.v_head + e0, x);
        store_chunk<T, kAligned>(stored_v + g * a.v_cache_head + e0, x);
      }
      continue;
    }
    const bool is_q = h < a.heads;
    const int g = is_q ? h : h - a.heads;
    if (mine) load_chunk<T, kAligned>(is_q ? static_cast<const T*>(a.q) + t * a.q_row + g * a.q_head + e0 : static_cast<const T*>(a.k) + t * a.k_row + g * a.k_head + e0, x);
    const void* weight = is_q ? a.q_weight : a.k_weight;
    if (weight) {
      float squares = 0;
      if (mine) {
#pragma unroll
        for (int i = 0; i < C; ++i) squares += x[i] * x[i];
      }
      for (int o = width >> 1; o >= 1; o >>= 1) squares += __shfl_xor(squares, o, kWave);
      const float inverse = rsqrtf(squares / a.dim + a.eps);
      if (mine) {
        float w[C];
        load_weight<T>(weight, a.weights32, e0, w);
#pragma unroll
        for (int i = 0; i < C; ++i) x[i] *= inverse * w[i];
      }
    }
    if (a.interleaved) {
      if (turned) {
#pragma unroll
        for (int i = 0; i < C; i += 2) {
          const float u = x[i], w = x[i + 1];
          x[i] = u * cosine[i] - w * sine[i];
          x[i + 1] = u * sine[i] + w * cosine[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const float other = __shfl(x[i], partner, kWave);
        if (turned) x[i] = e0 < half ? x[i] * cosine[i] - other * sine[i] : x[i] * cosine[i] + other * sine[i];
      }
    }
    if (!mine) continue;
    if (is_q) {
      store_chunk<T, kAligned>(static_cast<T*>(a.q_out) + t * a.q_out_row + g * a.q_out_head + e0, x);
    } else {
      if (a.k_out) store_chunk<T, kAligned>(static_cast<T*>(a.k_out) + t * a.k_out_row + g * a.k_out_head + e0, x);
      if (stored_k) store_chunk<T, kAligned>(stored_k + g * a.k_cache_head + e0, x);
    }
  }
}

bool aligned(const void* p, int64_t row, int64_t head, int64_t block, int size) {
  return !p || ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(row * size) | static_cast<uintptr_t>(head * size) | static_cast<uintptr_t>(block * size)) & 15) == 0;
}

template <typename T> void launch(const MloraRotateArgs& a) {
  constexpr int C = 16 / sizeof(T);
  int width = 1;
  while (width * C < a.dim) width *= 2;
  const int all = a.heads + a.kv_heads + (a.v ? a.kv_heads : 0);
  const int per = 1, chunks = (all + per - 1) / per;
  const long long units = static_cast<long long>(a.num_tokens) * chunks;
  const unsigned grid = static_cast<unsigned>((units * width + kThreads - 1) / kThreads);
  const int size = sizeof(T);
  const bool vectors = aligned(a.q, a.q_row, a.q_head, 0, size) && aligned(a.k, a.k_row, a.k_head, 0, size) && aligned(a.v, a.v_row, a.v_head, 0, size) &&
                       aligned(a.q_out, a.q_out_row, a.q_out_head, 0, size) && aligned(a.k_out, a.k_out_row, a.k_out_head, 0, size) &&
                       aligned(a.k_cache, a.k_cache_row, a.k_cache_head, a.k_block, size) && aligned(a.v_cache, a.v_cache_row, a.v_cache_head, a.v_block, size);
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  if (vectors) rotate_kernel<T, true><<<grid, kThreads, 0, stream>>>(a, width, per, chunks);
  else rotate_kernel<T, false><<<grid, kThreads, 0, stream>>>(a, width, per, chunks);
}

}  // namespace

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_rotate_qk(const MloraRotateArgs* a) {
  if (!a) { set_error("mlora_rotate_qk: NULL args"); return MLORA_E_INVALID; }
  if (a->num_tokens < 0 || a->heads < 0 || a->kv_heads < 0 || a->num_blocks < 0 || a->num_positions < 0) {
    set_error("mlora_rotate_qk: negative size");
    return MLORA_E_INVALID;
  }
  if (a->dtype != MLORA_DTYPE_F32 && a->dtype != MLORA_DTYPE_F16 && a->dtype != MLORA_DTYPE_BF16) {
    set_error("mlora_rotate_qk: unknown dtype %d", a->dtype);
    return MLORA_E_INVALID;
  }
  if (a->dim < 8 || a->dim % 8 || a->dim > MLORA_MAX_HEAD_DIM) {
    set_error("mlora_rotate_qk: dim = %d is not a multiple of 8 up to %d", a->dim, MLORA_MAX_HEAD_DIM);
    return MLORA_E_UNSUPPORTED;
  }
  if (a->rotary < 0 || a->rotary % 16 || a->rotary > a->dim) {
    set_error("mlora_rotate_qk: rotary = %d is not a multiple of 16 up to dim = %d", a->rotary, a->dim);
    return MLORA_E_UNSUPPORTED;
  }
  if (a->num_tokens == 0 || a->heads + static_cast<int64_t>(a->kv_heads) == 0) return 0;
  if (!a->positions || (a->rotary && !a->cos_sin) || (a->heads && (!a->q || !a->q_out)) || (a->kv_heads && !a->k)) {
    set_error("mlora_rotate_qk: NULL pointer");
    return MLORA_E_INVALID;
  }
  if ((a->k_cache || a->v_cache || a->slots) && (!a->k_cache || !a->v_cache || !a->slots || !a->v || a->page < 1)) {
    set_error("mlora_rotate_qk: a cache needs k_cache, v_cache, v, slots and a page of at least one row");
    return MLORA_E_INVALID;
  }
  if (a->v && !a->slots) { set_error("mlora_rotate_qk: v is stored only: it needs a cache"); return MLORA_E_INVALID; }
  const int64_t all = static_cast<int64_t>(a->heads) + 2 * static_cast<int64_t>(a->kv_heads);
  if (all * a->num_tokens > (1ll << 30)) { set_error("mlora_rotate_qk: %d tokens of %d + %d heads are more than one launch holds", a->num_tokens, a->heads, a->kv_heads); return MLORA_E_TOO_LARGE; }
  if (a->dtype == MLORA_DTYPE_BF16) launch<__bf16>(*a);
  else if (a->dtype == MLORA_DTYPE_F16) launch<_Float16>(*a);
  else launch<float>(*a);
  return check_launch("mlora_rotate_qk");
}
