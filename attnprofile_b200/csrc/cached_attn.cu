// attn_cached: argument checks and the choice of kernels.
#include "cached_attn.cuh"

#include <cmath>

using namespace attnprof::cache;

namespace {
int capacity_of(int width, int block_size) {
  const long long n = static_cast<long long>(width) * block_size;
  return n > INT_MAX - 4096 ? INT_MAX - 4096 : static_cast<int>(n);
}

// Rows of one request and kv head up to which the split kernel is used, above
// it the tiled one.  Measured in graphs, both ways (8 kv heads, e4m3; split |
// tiled, us): D = 64, 32 rows: 8 requests of 4000 tokens 32 | 41, 2 of 30,000
// 34 | 55; 48 rows: 44 | 39, 69 | 55.  D = 128, 16 rows: 24 | 44, 36 | 69; 24
// rows: 47 | 45, 67 | 69, 64 requests of 1000 tokens 102 | 90.
constexpr long long split_rows(int D) { return D == 64 ? 32 : 16; }
}  // namespace

extern "C" int attn_cached(const attn_cached_args* args, void* stream) {
  if (!args) return ATTN_ERR_INVALID_ARG;
  const attn_cached_args& a = *args;
  const int rc = check_pool(a.num_blocks, a.kv_heads, a.block_size, a.D, a.code);
  if (rc != ATTN_OK) return rc;
  if (!dtype_ok(a.dtype)) return ATTN_ERR_UNSUPPORTED;
  if (a.tokens < 0 || a.batch < 0 || a.max_new < 0 || a.width < 0 || a.heads <= 0 ||
      a.heads % a.kv_heads != 0 || a.table_stride < a.width || !std::isfinite(a.scale) ||
      a.scale < 0.f)
    return ATTN_ERR_INVALID_ARG;
  if (a.tokens == 0 || a.batch == 0 || a.max_new == 0) return ATTN_OK;
  if (!a.q || !a.out || !a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale || !a.kv_lens ||
      !a.starts || (a.width > 0 && !a.tables))
    return ATTN_ERR_INVALID_ARG;
  // Rows that would be written over each other, or read after they were written.
  if ((a.tokens > 1 && a.out_token_stride == 0) || (a.heads > 1 && a.out_head_stride == 0) ||
      a.q == a.out)
    return ATTN_ERR_INVALID_ARG;
  if (!aligned(a.q, 16) || !aligned(a.out, 16) || !aligned(a.k_codes, 16) ||
      !aligned(a.v_codes, 16) || !aligned(a.workspace, 16) || !aligned(a.k_scale, 4) ||
      !aligned(a.v_scale, 4) || !aligned(a.tables, 4) || !aligned(a.kv_lens, 4) ||
      !aligned(a.starts, 4) ||
      ((a.q_token_stride | a.q_head_stride | a.out_token_stride | a.out_head_stride) & 7) != 0)
    return ATTN_ERR_MISALIGNED;
  const int group = a.heads / a.kv_heads;
  const long long most = static_cast<long long>(a.max_new) * group;  // rows of a request and kv head
  if (most > INT_MAX) return ATTN_ERR_INVALID_ARG;
  CachedParams p{};
  p.q = a.q;
  p.out = a.out;
  p.kc = static_cast<const uint8_t*>(a.k_codes);
  p.vc = static_cast<const uint8_t*>(a.v_codes);
  p.ks = a.k_scale;
  p.vs = a.v_scale;
  p.tables = a.tables;
  p.kv_lens = a.kv_lens;
  p.starts = a.starts;
  p.q_token = a.q_token_stride;
  p.q_head = a.q_head_stride;
  p.o_token = a.out_token_stride;
  p.o_head = a.out_head_stride;
  p.table_stride = a.table_stride;
  p.tokens = a.tokens;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.group = group;
  p.batch = a.batch;
  p.max_new = a.max_new;
  p.num_blocks = a.num_blocks;
  p.shift = shift_of(a.block_size);
  p.capacity = capacity_of(a.width, a.block_size);
  p.causal = a.causal != 0;
  p.scale_log2 = static_cast<float>(
      (a.scale > 0.f ? static_cast<double>(a.scale) : 1.0 / std::sqrt(static_cast<double>(a.D))) *
      1.4426950408889634);
  // A batch may hold requests for both kernels (the lengths are on the GPU): then both run,
  // each on its own requests.  A single request, or none that can be long,
  // needs one launch.
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (most <= split_rows(a.D)) {
    p.rows_most = LLONG_MAX;
  } else {
    const bool tiled_only = a.batch == 1 || group > split_rows(a.D);
    p.rows_most = tiled_only ? 0 : split_rows(a.D);
    const int rt = launch_tiled(p, a.D, a.dtype, a.code, a.workspace, a.workspace_bytes, st);
    if (rt != ATTN_OK || tiled_only) return rt;
  }
  return launch_split(p, a.D, a.dtype, a.code, a.max_new, a.workspace, a.workspace_bytes, st);
}

extern "C" int attn_cached_workspace(int heads, int kv_heads, int D, int max_new, int block_size,
                                     int width, unsigned long long* bytes) {
  if (!bytes || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || max_new < 0 || width < 0)
    return ATTN_ERR_INVALID_ARG;
  if ((D != 64 && D != 128) || !block_size_ok(block_size)) return ATTN_ERR_UNSUPPORTED;
  const int group = heads / kv_heads, capacity = capacity_of(width, block_size);
  const int rows = max_new > 0 ? max_new : 1;
  int rc = split_workspace(group, D, rows, capacity, bytes);
  if (rc == ATTN_OK && static_cast<long long>(rows) * group > split_rows(D)) {
    unsigned long long tiled = 0;
    rc = tiled_workspace(D, capacity, &tiled);
    if (rc == ATTN_OK && tiled > *bytes) *bytes = tiled;
  }
  return rc;
}
