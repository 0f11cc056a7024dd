// What the kernels of attention.hip share: where a query row stands, which keys it sees and where those lie.
#pragma once
#include "common.h"
#include "mlora.h"

namespace mlora {

// attention.hip
bool attention_vectors_ok(const MloraAttentionArgs* a);  // every row of q, out, k and v starts on a 16-byte boundary
int launch_attend_rows(const MloraAttentionArgs* a);     // any head size, stride and page

// paged.hip: one row per sequence over pages, head sizes 64 and 128
bool paged_supported(const MloraAttentionArgs* a);
size_t paged_workspace_bytes(const MloraAttentionArgs* a);
int launch_paged(const MloraAttentionArgs* a);

// prompt.hip: packed rows, head sizes 64 and 128
bool prompt_supported(const MloraAttentionArgs* a);
size_t prompt_workspace_bytes(const MloraAttentionArgs* a);
int launch_prompt(const MloraAttentionArgs* a);

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// The keys that a query at position p of a sequence of `total` keys sees: [0, first) and [low, high).
struct Visible {
  int first, low, high;
  __device__ __forceinline__ int count() const { return first + high - low; }
  __device__ __forceinline__ int key(int i) const { return i < first ? i : i - first + low; }
};
__device__ __forceinline__ Visible visible_keys(const MloraAttentionArgs& a, int p, int total) {
  Visible v;
  v.high = a.causal && p + 1 < total ? (p + 1 > 0 ? p + 1 : 0) : total;
  v.low = a.window && v.high > a.window ? v.high - a.window : 0;
  v.first = a.sinks < v.low ? a.sinks : v.low;
  return v;
}

// A sequence of the batch: its keys, and where its query rows start.  Whatever the device's vectors hold, rows stay inside q and keys inside k or the table.
struct Place {
  int sequence, total, key_start, position;  // position: of the row that was asked for
};
__device__ __forceinline__ int clamped(int v, int most) { return v < 0 ? 0 : v > most ? most : v; }
__device__ __forceinline__ int keys_of(const MloraAttentionArgs& a, int s, int* key_start) {
  if (a.block_tables) {
    *key_start = 0;
    return clamped(a.context_lens[s], a.table_width * a.page);
  }
  const int32_t* starts = a.key_starts ? a.key_starts : a.starts;
  const int begin = clamped(starts[s], a.num_keys), end = clamped(starts[s + 1], a.num_keys);
  *key_start = begin;
  return end > begin ? end - begin : 0;
}
// False for a row in front of the first sequence or behind the last.
__device__ __forceinline__ bool place_of_row(const MloraAttentionArgs& a, int row, Place* at) {
  if (!a.starts) {  // a row per sequence
    at->sequence = row;
    at->total = keys_of(a, row, &at->key_start);
    at->position = at->total - 1;
    return true;
  }
  if (row < a.starts[0] || row >= a.starts[a.sequences]) return false;
  int lo = 0, hi = a.sequences;  // starts[lo] <= row < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  at->sequence = lo;
  at->total = keys_of(a, lo, &at->key_start);
  at->position = at->total - (a.starts[lo + 1] - row);
  return true;
}

// Row of a key (strides in elements), nullptr for one of a page outside the cache.
template <typename T> struct KeyRow {
  const T* k;
  const T* v;
};
template <typename T> __device__ __forceinline__ KeyRow<T> key_row(const MloraAttentionArgs& a, const Place& at, int kv_head, int key) {
  KeyRow<T> r{nullptr, nullptr};
  if (a.block_tables) {
    const int page = key / a.page, in_page = key - page * a.page;
    const int block = a.block_tables[at.sequence * a.table_row + page];
    if (block < 0 || block >= a.num_blocks) return r;
    r.k = static_cast<const T*>(a.k) + block * a.k_block + in_page * a.k_row + kv_head * a.k_head;
    r.v = static_cast<const T*>(a.v) + block * a.v_block + in_page * a.v_row + kv_head * a.v_head;
  } else {
    r.k = static_cast<const T*>(a.k) + (at.key_start + key) * a.k_row + kv_head * a.k_head;
    r.v = static_cast<const T*>(a.v) + (at.key_start + key) * a.v_row + kv_head * a.v_head;
  }
  return r;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
  return v;
}

// One (query row, head) by one wavefront; `query`: MLORA_MAX_HEAD_DIM floats of LDS of its own.
template <typename T> __device__ void attend_row(const MloraAttentionArgs& a, const Place& at, int row, int head, int lane, float* query) {
  constexpr int kParts = MLORA_MAX_HEAD_DIM / 64;
  const T* q = static_cast<const T*>(a.q) + row * a.q_row + head * a.q_head;
  for (int e = lane; e < a.dim; e += 64) query[e] = to_f32(q[e]) * (a.scale * kLog2e);
  __builtin_amdgcn_wave_barrier();
  const Visible seen = visible_keys(a, at.position, at.total);
  const int count = seen.count();
  const int kv_head = head / (a.heads / a.kv_heads);
  float m = -__builtin_inff(), l = 0.0f, o[kParts] = {};
  bool any = false;
  for (int base = 0; base < count; base += 64) {
    const int n = count - base < 64 ? count - base : 64;
    KeyRow<T> r{nullptr, nullptr};
    float s = -__builtin_inff();
    if (lane < n) r = key_row<T>(a, at, kv_head, seen.key(base + lane));
    if (r.k) {
      s = 0.0f;
      for (int e = 0; e < a.dim; ++e) s += query[e] * to_f32(r.k[e]);
    }
    const unsigned long long there = __ballot(r.k != nullptr);
    any |= there != 0;
    // (a score that is NaN makes m stay and p NaN; with nothing but -inf so far the base is 0)
    const float top = fmaxf(m, wave_max(s)), base2 = top == -__builtin_inff() ? 0.0f : top;
    const float alpha = exp2f(m - base2), p = exp2f(s - base2);
    m = top;
    l = l * alpha + wave_sum(r.k ? p : 0.0f);
#pragma unroll
    for (int i = 0; i < kParts; ++i) o[i] *= alpha;
    for (int j = 0; j < n; ++j) {
      if (!(there >> j & 1)) continue;
      const float pj = __shfl(p, j, kWave);
      const T* v = reinterpret_cast<const T*>(__shfl(static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(r.v)), j, kWave));
#pragma unroll
      for (int i = 0; i < kParts; ++i)
        if (lane + 64 * i < a.dim) o[i] += pj * to_f32(v[lane + 64 * i]);
    }
  }
  T* out = static_cast<T*>(a.out) + row * a.out_row + head * a.out_head;
#pragma unroll
  for (int i = 0; i < kParts; ++i)
    if (lane + 64 * i < a.dim) out[lane + 64 * i] = from_f32<T>(any ? o[i] / l : 0.0f);
}

}  // namespace

}  // namespace mlora
