// Norm, rotation and cache store of a batch's query, key and value heads (mlora_rotate_qk); stands where the reference turns them and
// stores keys and values in its cache (nanovllm_voxcpm/layers/rotary_embedding.py, layers/attention.py:10-50).
//
// A head is W lanes of 16 bytes each (W = dim / 8, in fp32 dim / 4, up to the next power of two): its mean square is a butterfly over
// those lanes, and what an element is paired with comes from the lane W / 2 on (or, in neighbouring pairs, from the lane itself).  With the weights taken into the
// cosines and sines an element is inverse * (own * x + paired * other): all of it in fp32, one rounding at the end.
//
// Bound by memory: a batch's heads are read once and written once.  A group of W lanes takes four heads of one token, for which it holds the coefficients in
// registers: read anew for every head they would be as many bytes as the head again.  9392 tokens, 16 + 2 heads of 64, bf16, norms and cache: 13.0 us,
// 3.7 TB/s (an elementwise operation over as many bytes 9.2 us: what is more here is the trip from positions to the table and the arithmetic of norm and rotation);
// 8381 tokens, 32 + 8 heads of 128, fp16: 41.9 us, 4.9 TB/s (39).
#include "common.h"
#include "launch.h"

namespace mlora {

namespace {

constexpr int kThreads = 256;
constexpr long long kManyThreads = 256 * 2048;  // of groups of one head: as many as the chip holds at once

// 16 bytes of a head.
template <typename T> struct Piece {
  static constexpr int C = 16 / sizeof(T);
  i32x4 raw;
  template <bool kAligned> __device__ __forceinline__ void load(const T* p) {
    if constexpr (kAligned) {
      raw = load128(p);
    } else {
      T e[C];
#pragma unroll
      for (int i = 0; i < C; ++i) e[i] = p[i];
      __builtin_memcpy(&raw, e, 16);
    }
  }
  template <bool kAligned> __device__ __forceinline__ void store(T* p) const {
    if constexpr (kAligned) {
      store128(p, raw);
    } else {
      T e[C];
      __builtin_memcpy(e, &raw, 16);
#pragma unroll
      for (int i = 0; i < C; ++i) p[i] = e[i];
    }
  }
  __device__ __forceinline__ void unpack(float (&x)[C]) const {
    if constexpr (C == 8) {
      Pack8 p;
      p.raw = raw;
      unpack8<T>(p, x);
    } else {
      __builtin_memcpy(x, &raw, 16);
    }
  }
  __device__ __forceinline__ void pack(const float (&x)[C]) {
    if constexpr (C == 8) {
      Pack8 p;
      pack8<T>(x, p);
      raw = p.raw;
    } else {
      __builtin_memcpy(&raw, x, 16);
    }
  }
};

// Sum over the `width` lanes of a head (a power of two), in every one of them.  Up to 16 lanes without LDS: neighbours, then neighbours' neighbours,
// then the mirrored half row and row, whose lanes hold the same sums by then.
template <int kControl> __device__ __forceinline__ float moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kControl, 0xf, 0xf, true));
}
__device__ __forceinline__ float head_sum(float v, int width) {
  if (width > 1) v += moved<0xb1>(v);
  if (width > 2) v += moved<0x4e>(v);
  if (width > 4) v += moved<0x141>(v);
  if (width > 8) v += moved<0x140>(v);
  for (int o = 16; o < width; o <<= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// `count` floats from p on (where kAligned: 16-byte aligned, `count` a multiple of four).
template <int kCount, bool kAligned> __device__ __forceinline__ void load_floats(const float* p, float* out) {
  if constexpr (kAligned) {
#pragma unroll
    for (int i = 0; i < kCount; i += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[i + j] = v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i) out[i] = p[i];
  }
}

template <typename T, bool kAligned> __device__ __forceinline__ void load_weight(const void* w, bool weights32, int at, float (&out)[16 / sizeof(T)]) {
  if (weights32) {
    load_floats<16 / static_cast<int>(sizeof(T)), kAligned>(static_cast<const float*>(w) + at, out);
  } else {
    Piece<T> p;
    p.template load<kAligned>(static_cast<const T*>(w) + at);
    p.unpack(out);
  }
}

// 16 bytes of lane ^ kDistance (a power of two up to 8), without LDS.
template <int kDistance> __device__ __forceinline__ i32x4 across(i32x4 v) {
  i32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x = __int_as_float(v[j]);
    if constexpr (kDistance == 1) x = moved<0xb1>(x);
    else if constexpr (kDistance == 2) x = moved<0x4e>(x);
    else if constexpr (kDistance == 4) x = moved<0x1b>(moved<0x141>(x));  // (i ^ 7) ^ 3
    else x = moved<0x141>(moved<0x140>(x));                               // (i ^ 15) ^ 7
    r[j] = __float_as_int(x);
  }
  return r;
}
template <int kDistance, typename T, int N> __device__ __forceinline__ void all_across(const Piece<T> (&x)[N], Piece<T> (&other)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) other[i].raw = across<kDistance>(x[i].raw);
}

// Groups of a token and how a number is divided by them: n / d = (n magic >> 32) >> shift for n below 2^31, with magic = 2^(31 + L) / d + 1, L = the
// bits of d - 1 and shift = L - 1; d of one has no such number.
struct Groups {
  int count, shift;
  uint32_t magic;
  Groups(int heads, int per) : count((heads + per - 1) / per) {
    int bits = 1;
    while ((1u << bits) < static_cast<unsigned>(count)) ++bits;
    shift = bits - 1;
    magic = count ? static_cast<uint32_t>((1ull << (31 + bits)) / count + 1) : 0;
  }
};

// A workgroup has heads of one kind, which so costs its wavefronts no choice lane by lane: the first `q_blocks` those of q, the next `kv_blocks` those
// of k, the rest those of v.
struct Layout {
  int log_width;  // lanes of a head
  unsigned q_blocks, kv_blocks;
  Groups q, kv;
  float inverse_dim;  // 1 / dim
};

// kPer: heads of a group.
template <typename T, bool kAligned, int kPer, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rotate_kernel(MloraRotateArgs a, Layout layout) {
  constexpr int C = 16 / sizeof(T);
  const int lane = threadIdx.x & 63, c = lane & ((1 << layout.log_width) - 1);
  const bool is_q = blockIdx.x < layout.q_blocks, is_v = blockIdx.x >= layout.q_blocks + layout.kv_blocks;
  const unsigned block_of_kind = blockIdx.x - (is_q ? 0 : layout.q_blocks + (is_v ? layout.kv_blocks : 0));
  const Groups& groups = is_q ? layout.q : layout.kv;
  const unsigned unit = (block_of_kind * kThreads + threadIdx.x) >> layout.log_width;
  const int t = groups.count == 1 ? unit : __umulhi(unit, groups.magic) >> groups.shift, group = unit - t * groups.count;
  if (t >= a.num_tokens) return;
  const int e0 = c * C, half = a.rotary >> 1;
  const bool mine = e0 < a.dim;
  const int first = group * kPer, heads = is_q ? a.heads : a.kv_heads;
  const bool turned = e0 < a.rotary && !is_v;
  const int partner = e0 < half ? e0 + half : e0 - half;  // first element of the other halves of this lane's pairs
  const int64_t head_stride = is_q ? a.q_head : is_v ? a.v_head : a.k_head, row_stride = is_q ? a.q_row : is_v ? a.v_row : a.k_row;
  const T* from = static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) + t * row_stride + first * head_stride;

  // every head's elements, and the ones they are paired with
  Piece<T> x[kPer], other[kPer];
  const T* at = from + e0;
#pragma unroll
  for (int i = 0; i < kPer; ++i, at += head_stride)
    if (first + i < heads && mine) x[i].template load<kAligned>(at);
  const int distance = half / C;  // between the lanes of a pair
  const bool exchange = kAligned && (distance == 1 || distance == 2 || distance == 4 || distance == 8);
  if (!kInterleaved && turned && !exchange) {
    at = from + partner;
#pragma unroll
    for (int i = 0; i < kPer; ++i, at += head_stride)
      if (first + i < heads) other[i].template load<kAligned>(at);
  }

  int64_t position = 0, slot = -1;
  if (turned) position = a.positions64 ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int32_t*>(a.positions)[t];
  if (a.slots && !is_q) slot = a.slots64 ? static_cast<const int64_t*>(a.slots)[t] : static_cast<const int32_t*>(a.slots)[t];

  // An element comes out as inverse * (own * x + paired * other), the weights taken into the cosines and sines.
  const void* weights = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
  float own[C], paired[C];
  if (turned) {
    constexpr int P = kInterleaved ? C / 2 : C;
    float cosine[P], sine[P];
    if (position >= 0 && position < a.num_positions) {
      const float* row = a.cos_sin + position * a.table_row + (kInterleaved ? e0 >> 1 : e0 < half ? e0 : e0 - half);
      load_floats<P, kAligned && P >= 4>(row, cosine);
      load_floats<P, kAligned && P >= 4>(row + half, sine);
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) cosine[i] = sine[i] = __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      own[i] = cosine[kInterleaved ? i >> 1 : i];
      paired[i] = sine[kInterleaved ? i >> 1 : i];
      if (kInterleaved ? !(i & 1) : e0 < half) paired[i] = -paired[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      own[i] = 1.0f;
      paired[i] = 0.0f;
    }
  }
  if (weights && mine) {
    float w[C];
    load_weight<T, kAligned>(weights, a.weights32, e0, w);
#pragma unroll
    for (int i = 0; i < C; ++i) own[i] *= w[i];
    if constexpr (kInterleaved) {
#pragma unroll
      for (int i = 0; i < C; ++i) paired[i] *= w[i ^ 1];
    } else if (turned) {
      load_weight<T, kAligned>(weights, a.weights32, partner, w);
#pragma unroll
      for (int i = 0; i < C; ++i) paired[i] *= w[i];
    }
  }
  if (!kInterleaved && exchange) {
    if (distance == 1) all_across<1>(x, other);
    else if (distance == 2) all_across<2>(x, other);
    else if (distance == 4) all_across<4>(x, other);
    else all_across<8>(x, other);
  }
  if (!kInterleaved && !turned) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) other[i].raw = i32x4{0, 0, 0, 0};
  }

  // where they go: q to q_out; k to k_out and the cache, v to the cache
  T* out = static_cast<T*>(is_q ? a.q_out : is_v ? nullptr : a.k_out);
  T* stored = nullptr;
  const int64_t out_stride = is_q ? a.q_out_head : a.k_out_head, stored_stride = is_v ? a.v_cache_head : a.k_cache_head;
  if (out) out += t * (is_q ? a.q_out_row : a.k_out_row) + first * out_stride + e0;
  if (slot >= 0 && slot < static_cast<int64_t>(a.num_blocks) * a.page) {
    // (slots of 32 bits are divided in 32)
    const int64_t block = slot <= UINT32_MAX ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.page) : slot / a.page, row = slot - block * a.page;
    stored = static_cast<T*>(is_v ? a.v_cache : a.k_cache) + block * (is_v ? a.v_block : a.k_block) + row * (is_v ? a.v_cache_row : a.k_cache_row) +
             first * stored_stride + e0;
  }

#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    float y[C];
    x[i].unpack(y);
    float inverse = 1.0f;
    if (weights) {
      float squares = 0;
#pragma unroll
      for (int j = 0; j < C; ++j) squares += y[j] * y[j];
      inverse = rsqrtf(head_sum(mine ? squares : 0.0f, 1 << layout.log_width) * layout.inverse_dim + a.eps);
    }
    if (!is_v) {
      float z[C];
      if constexpr (kInterleaved) {
#pragma unroll
        for (int j = 0; j < C; ++j) z[j] = turned ? y[j ^ 1] : 0.0f;
      } else {
        other[i].unpack(z);
      }
#pragma unroll
      for (int j = 0; j < C; ++j) y[j] = (y[j] * own[j] + z[j] * paired[j]) * inverse;
      x[i].pack(y);
    }
    if (first + i >= heads || !mine) continue;
    if (out) x[i].template store<kAligned>(out + i * out_stride);
    if (stored) x[i].template store<kAligned>(stored + i * stored_stride);
  }
}

bool aligned(const void* p, int64_t row, int64_t head, int64_t block, int size) {
  return !p || ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(row * size) | static_cast<uintptr_t>(head * size) | static_cast<uintptr_t>(block * size)) & 15) == 0;
}

template <typename T, bool kAligned, int kPer> void launch_heads(const MloraRotateArgs& a, int log_width) {
  const Groups q(a.heads, kPer), kv(a.kv_heads, kPer);
  auto blocks = [&](int groups) { return static_cast<unsigned>((((static_cast<long long>(a.num_tokens) * groups) << log_width) + kThreads - 1) / kThreads); };
  const Layout layout{log_width, blocks(q.count), blocks(kv.count), q, kv, 1.0f / a.dim};
  const unsigned grid = layout.q_blocks + layout.kv_blocks * (a.v ? 2 : 1);
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  if (a.interleaved) rotate_kernel<T, kAligned, kPer, true><<<grid, kThreads, 0, stream>>>(a, layout);
  else rotate_kernel<T, kAligned, kPer, false><<<grid, kThreads, 0, stream>>>(a, layout);
}

template <typename T> void launch(const MloraRotateArgs& a) {
  constexpr int C = 16 / sizeof(T);
  int log_width = 0;
  while ((C << log_width) < a.dim) ++log_width;
  const int all = a.heads + a.kv_heads + (a.v ? a.kv_heads : 0), size = sizeof(T);
  const bool vectors = aligned(a.q, a.q_row, a.q_head, 0, size) && aligned(a.k, a.k_row, a.k_head, 0, size) && aligned(a.v, a.v_row, a.v_head, 0, size) &&
                       aligned(a.q_out, a.q_out_row, a.q_out_head, 0, size) && aligned(a.k_out, a.k_out_row, a.k_out_head, 0, size) &&
                       aligned(a.k_cache, a.k_cache_row, a.k_cache_head, a.k_block, size) && aligned(a.v_cache, a.v_cache_row, a.v_cache_head, a.v_block, size) &&
                       aligned(a.cos_sin, a.table_row, 0, 0, 4) && aligned(a.q_weight, 0, 0, 0, 1) && aligned(a.k_weight, 0, 0, 0, 1);
  // Four heads a group read the table and the weights a fourth as often as one (9392 tokens, 16 + 2 heads of 64, bf16, norms: 1, 2, 4, 8 heads 15.7, 14.1,
  // 13.0, 14.2 us; 8381, 32 + 8 of 128, fp16: 52.0, 42.4, 41.9, 42.8); with few tokens one, so that every compute unit has some.
  const bool many = (static_cast<long long>(a.num_tokens) * all << log_width) >= kManyThreads;
  if (!vectors) launch_heads<T, false, 1>(a, log_width);
  else if (many) launch_heads<T, true, 4>(a, log_width);
  else launch_heads<T, true, 1>(a, log_width);
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
  if (all * a->num_tokens > (1ll << 25)) { set_error("mlora_rotate_qk: %d tokens of %d + %d heads are more than one launch holds", a->num_tokens, a->heads, a->kv_heads); return MLORA_E_TOO_LARGE; }
  if (a->dtype == MLORA_DTYPE_BF16) launch<__bf16>(*a);
  else if (a->dtype == MLORA_DTYPE_F16) launch<_Float16>(*a);
  else launch<float>(*a);
  return check_launch("mlora_rotate_qk");
}
