// attn_cached: argument checks and the choice of kernels.
#include "cached_attn.cuh"

#include <cmath>

using namespace attnprof::cache;

namespace {
constexpr long long kSplitRows = 64;
}

extern "C" int attn_cached(const void* q, long long q_token_stride, long long q_head_stride,
                           void* out, long long out_token_stride, long long out_head_stride,
                           int tokens, int heads, int kv_heads, int D, int dtype,
                           const void* k_codes, const void* v_codes, const float* k_scale,
                           const float* v_scale, int code, int num_blocks, int block_size,
                           const int* tables, int width, long long table_stride,
                           const int* kv_lens, const int* starts, int batch, int max_new,
                           int causal, float scale, void* workspace,
                           unsigned long long workspace_bytes, void* stream) {
  const int rc = check_pool(num_blocks, kv_heads, block_size, D, code);
  if (rc != ATTN_OK) return rc;
  if (!dtype_ok(dtype)) return ATTN_ERR_UNSUPPORTED;
  if (tokens < 0 || batch < 0 || max_new < 0 || width < 0 || heads <= 0 || heads % kv_heads != 0 ||
      table_stride < width || !std::isfinite(scale) || scale < 0.f)
    return ATTN_ERR_INVALID_ARG;
  if (tokens == 0 || batch == 0 || max_new == 0) return ATTN_OK;
  if (!q || !out || !k_codes || !v_codes || !k_scale || !v_scale || !kv_lens || !starts ||
      !workspace || (width > 0 && !tables))
    return ATTN_ERR_INVALID_ARG;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_codes, 16) || !aligned(v_codes, 16) ||
      !aligned(workspace, 16) ||
      ((q_token_stride | q_head_stride | out_token_stride | out_head_stride) & 7) != 0)
    return ATTN_ERR_MISALIGNED;
  if (static_cast<long long>(max_new) * (heads / kv_heads) > INT_MAX) return ATTN_ERR_INVALID_ARG;
  CachedParams p{};
  p.q = q;
  p.out = out;
  p.kc = static_cast<const uint8_t*>(k_codes);
  p.vc = static_cast<const uint8_t*>(v_codes);
  p.ks = k_scale;
  p.vs = v_scale;
  p.tables = tables;
  p.kv_lens = kv_lens;
  p.starts = starts;
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.o_token = out_token_stride;
  p.o_head = out_head_stride;
  p.table_stride = table_stride;
  p.tokens = tokens;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.batch = batch;
  p.num_blocks = num_blocks;
  p.shift = block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
  const long long capacity = static_cast<long long>(width) * block_size;
  p.capacity = capacity > INT_MAX - 4096 ? INT_MAX - 4096 : static_cast<int>(capacity);
  p.causal = causal != 0;
  p.scale_log2 = static_cast<float>(
      (scale > 0.f ? static_cast<double>(scale) : 1.0 / std::sqrt(static_cast<double>(D))) *
      1.4426950408889634);
  // Rows of one request and kv head: up to kSplitRows the keys' bytes are what
  // counts and the split kernel reads them with every SM; above, the tiled one.
  // A batch may hold both kinds (the lengths are on the GPU): then both run,
  // each on its own requests.  A single request, or none that can be long,
  // needs one launch.
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long most = static_cast<long long>(max_new) * p.group;
  if (most <= kSplitRows) {
    p.rows_most = LLONG_MAX;
    return launch_split(p, D, dtype, code, max_new, workspace, workspace_bytes, st);
  }
  p.rows_most = batch == 1 ? 0 : kSplitRows;
  const int rt = launch_tiled(p, D, dtype, code, st);
  if (rt != ATTN_OK || batch == 1) return rt;
  return launch_split(p, D, dtype, code, max_new, workspace, workspace_bytes, st);
}

extern "C" int attn_cached_workspace(int heads, int kv_heads, int D, int max_new,
                                     unsigned long long* bytes) {
  if (!bytes || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || max_new < 0)
    return ATTN_ERR_INVALID_ARG;
  if (D != 64 && D != 128) return ATTN_ERR_UNSUPPORTED;
  return split_workspace(heads / kv_heads, D, max_new > 0 ? max_new : 1, bytes);
}
