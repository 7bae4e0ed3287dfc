// Attention over the paged 8-bit cache: what its kernels share.
#pragma once

#include <cuda.h>

#include "cache.cuh"

namespace attnprof {
namespace cache {

struct CachedParams {
  const void* q;
  void* out;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *tables, *kv_lens, *starts;
  long long q_token, q_head, o_token, o_head, table_stride;
  int tokens, heads, kv_heads, group, batch, num_blocks, shift, capacity, causal;
  int whole;    // split kernel: no unit is cut
  int max_new;  // rows of a request at most
  float scale_log2;  // score scale * log2(e)
  // Requests of more than `rows_most` query rows a kv head (tokens * group)
  // belong to the other kernel: the split one takes those up to it, the tiled
  // one those above it.
  long long rows_most;
  float* ws;
};

// A request as the kernels see it, with every number brought into range.
struct Request {
  int start, n, kv;  // first query row, rows computed, tokens in the cache
  int before;        // tokens in front of the first row's own; negative: it has none
};

// FROM_L2: for the joining kernels, which ask before they wait for the kernel in
// front of them; only that wait makes L1 follow what was written since.  (L2 for
// all: 102 us where this took 91 on 64 requests of 5 to 8191 tokens.)
template <bool FROM_L2 = false>
__device__ __forceinline__ Request request_at(const CachedParams& p, int r) {
  auto load = [](const int* x) { return FROM_L2 ? __ldcg(x) : *x; };
  const int a = min(max(load(p.starts + r), 0), p.tokens);
  const int b = min(max(load(p.starts + r + 1), 0), p.tokens);
  const int rows = max(b - a, 0), kv = min(max(load(p.kv_lens + r), 0), p.capacity);
  // All rows count for what a row sees, those beyond max_new too.
  return Request{a, min(rows, p.max_new), kv, kv - rows};
}

int codes_map(CUtensorMap* m, const void* codes, const CachedParams& p, int D);
int launch_split(const CachedParams& p, int D, int dtype, int code, int max_new, void* ws,
                 unsigned long long ws_bytes, cudaStream_t st);
int launch_tiled(const CachedParams& p, int D, int dtype, int code, void* ws,
                 unsigned long long ws_bytes, cudaStream_t st);
int tiled_workspace(int D, int capacity, unsigned long long* bytes);
int split_workspace(int group, int D, int max_new, int capacity, unsigned long long* bytes);

}  // namespace cache
}  // namespace attnprof
