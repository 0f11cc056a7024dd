// Entry points of attention over paged or packed keys (mlora_decode_attention, mlora_prompt_attention; they stand where the
// reference calls its attention library, nanovllm_voxcpm/layers/attention.py:70-105), and the kernel that serves every shape:
// any head size, stride and page.
//
// One wavefront per (query row, head).  64 visible keys at a time, one per lane: the lane adds up its key's product with q (in LDS), the wave takes the
// running maximum m and sum l over, p = exp2(s - m), and the lanes, now elements of the head, add p_j v_j key by key:
// o <- o 2^(m_old - m) + sum_j p_j v_j, out = o / l.  Hidden keys are never enumerated, so nothing of them is read.
//
// It is right first of all, and bound by its own loads: element by element, a key per lane, nothing shared between heads, a sequence never split.  16 heads of 2 of 96, bf16: one stream of
// up to 900 keys 298 us, 64 of up to 2048 1245 us, 16 prompts of 587 2794 us; 3 streams of up to 131072, 8 heads of 96: 97 ms (head size 128 on the matrix cores 0.22).
#include "attention.h"
#include "common.h"
#include "launch.h"

namespace mlora {

namespace {

constexpr int kWaves = 4;
constexpr long long kLine = 1 << 20;  // workgroups along a launch's first dimension

template <typename T>
__global__ __launch_bounds__(kWaves * 64) void attend_rows_kernel(MloraAttentionArgs a) {
  __shared__ float queries[kWaves][MLORA_MAX_HEAD_DIM];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long unit = (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * kWaves + wave;
  const int row = static_cast<int>(unit / a.heads), head = static_cast<int>(unit - static_cast<long long>(row) * a.heads);
  if (unit >= static_cast<long long>(a.num_rows) * a.heads) return;
  Place at;
  if (!place_of_row(a, row, &at)) return;
  attend_row<T>(a, at, row, head, lane, queries[wave]);
}

}  // namespace

bool attention_vectors_ok(const MloraAttentionArgs* a) {
  const int size = a->dtype == MLORA_DTYPE_F32 ? 4 : 2;
  const uintptr_t rows = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v);
  int64_t strides = a->q_row | a->q_head | a->out_row | a->out_head | a->k_row | a->k_head | a->v_row | a->v_head;
  if (a->block_tables) strides |= a->k_block | a->v_block;
  return ((rows | static_cast<uintptr_t>(strides * size)) & 15) == 0;
}

int launch_attend_rows(const MloraAttentionArgs* a) {
  const long long units = static_cast<long long>(a->num_rows) * a->heads;
  // (a dimension of a launch has fewer than 2^32 threads: what is more goes along the second)
  const long long blocks = (units + kWaves - 1) / kWaves, line = blocks < kLine ? blocks : kLine;
  const dim3 grid(static_cast<unsigned>(line), static_cast<unsigned>((blocks + line - 1) / line));
  const hipStream_t stream = static_cast<hipStream_t>(a->stream);
  if (a->dtype == MLORA_DTYPE_BF16) attend_rows_kernel<__bf16><<<grid, kWaves * 64, 0, stream>>>(*a);
  else if (a->dtype == MLORA_DTYPE_F16) attend_rows_kernel<_Float16><<<grid, kWaves * 64, 0, stream>>>(*a);
  else attend_rows_kernel<float><<<grid, kWaves * 64, 0, stream>>>(*a);
  return check_launch("attention");
}

}  // namespace mlora

using namespace mlora;

namespace {

constexpr int kNothing = INT32_MIN;

int check_attention(const MloraAttentionArgs* a, const char* what, bool decode) {
  if (!a) { set_error("%s: NULL args", what); return MLORA_E_INVALID; }
  if (a->num_rows < 0 || a->num_keys < 0 || a->sequences < 0 || a->heads < 0 || a->kv_heads < 0 || a->table_width < 0 || a->num_blocks < 0 || a->window < 0 || a->sinks < 0) {
    set_error("%s: negative size", what);
    return MLORA_E_INVALID;
  }
  if (a->dtype != MLORA_DTYPE_F32 && a->dtype != MLORA_DTYPE_F16 && a->dtype != MLORA_DTYPE_BF16) {
    set_error("%s: unknown dtype %d", what, a->dtype);
    return MLORA_E_INVALID;
  }
  if (a->dim < 8 || a->dim % 8 || a->dim > MLORA_MAX_HEAD_DIM) {
    set_error("%s: dim = %d is not a multiple of 8 up to %d", what, a->dim, MLORA_MAX_HEAD_DIM);
    return MLORA_E_UNSUPPORTED;
  }
  if ((a->window || a->sinks) && !a->causal) { set_error("%s: a window or sinks need causal order", what); return MLORA_E_UNSUPPORTED; }
  if (a->num_rows == 0 || a->heads == 0 || a->sequences == 0) return kNothing;
  if (a->kv_heads == 0 || a->heads % a->kv_heads) { set_error("%s: %d heads do not share %d key-value heads evenly", what, a->heads, a->kv_heads); return MLORA_E_INVALID; }
  if (!a->q || !a->out) { set_error("%s: NULL pointer", what); return MLORA_E_INVALID; }
  if (decode) {
    if (!a->block_tables) { set_error("%s: keys lie in the pages of a cache: block_tables is NULL", what); return MLORA_E_INVALID; }
    if (a->num_rows != a->sequences) { set_error("%s: %d rows for %d sequences", what, a->num_rows, a->sequences); return MLORA_E_INVALID; }
    if (!a->causal) { set_error("%s: a new token has nothing behind it: causal must be set", what); return MLORA_E_INVALID; }
  } else if (!a->starts) {
    set_error("%s: starts is NULL", what);
    return MLORA_E_INVALID;
  }
  if (a->block_tables) {
    if (!a->context_lens || a->page < 1) { set_error("%s: pages need context_lens and a page of at least one row", what); return MLORA_E_INVALID; }
    if (static_cast<int64_t>(a->table_width) * a->page > INT32_MAX / 4) { set_error("%s: %d pages of %d rows are more positions than 2^29", what, a->table_width, a->page); return MLORA_E_TOO_LARGE; }
  }
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) { set_error("%s: workspace is not 16-byte aligned", what); return MLORA_E_INVALID; }
  const bool keys = a->block_tables ? a->num_blocks > 0 && a->table_width > 0 : a->num_keys > 0;
  if (keys && (!a->k || !a->v)) { set_error("%s: NULL pointer", what); return MLORA_E_INVALID; }
  if (static_cast<int64_t>(a->num_rows) * a->heads > (1ll << 30)) { set_error("%s: %d rows of %d heads are more than one launch holds", what, a->num_rows, a->heads); return MLORA_E_TOO_LARGE; }
  return 0;
}

}  // namespace

extern "C" int mlora_decode_attention(const MloraAttentionArgs* a) {
  const int rc = check_attention(a, "mlora_decode_attention", true);
  if (rc) return rc == kNothing ? 0 : rc;
  MloraAttentionArgs b = *a;
  b.starts = nullptr;
  if (paged_supported(&b)) return launch_paged(&b);
  return launch_attend_rows(&b);
}

// Blocks that the entry points would refuse need none.
static bool sized(const MloraAttentionArgs* a) {
  return a && a->num_rows > 0 && a->num_keys >= 0 && a->sequences > 0 && a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->dim > 0 &&
         a->table_width >= 0 && a->num_blocks >= 0 && a->page >= 0 && a->window >= 0 && a->sinks >= 0;
}

extern "C" size_t mlora_decode_attention_workspace_bytes(const MloraAttentionArgs* a) {
  return sized(a) && a->block_tables && a->page > 0 && paged_supported(a) ? paged_workspace_bytes(a) : 0;
}

extern "C" int mlora_prompt_attention(const MloraAttentionArgs* a) {
  const int rc = check_attention(a, "mlora_prompt_attention", false);
  if (rc) return rc == kNothing ? 0 : rc;
  if (prompt_supported(a)) return launch_prompt(a);
  return launch_attend_rows(a);
}

extern "C" size_t mlora_prompt_attention_workspace_bytes(const MloraAttentionArgs* a) { return sized(a) ? prompt_workspace_bytes(a) : 0; }
