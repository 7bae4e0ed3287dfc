// Block tables and slot maps on the GPU, from the requests' lengths.
//
// attn_block_tables gives every request the blocks that its new tokens need
// and writes each new token's slot; attn_block_trim takes back the blocks
// behind the tokens that a request keeps.  The pool's free blocks are a stack:
// free_blocks[0 .. free_count), taken from and returned to the top.
//
// The mathematics is two prefix sums over the requests (new tokens, blocks)
// and a search of them per token and per block.  It moves a few words a
// request and 4 bytes a token, so a call is bound by its launch and by the
// chain of loads, scan and stores (a few microseconds), not by bandwidth.
// Therefore one launch of one thread-block cluster: every CTA scans all
// requests into its own shared memory (that repeats a few KB of L2 reads,
// where a second launch or a global counter would cost more), a cluster
// barrier ends the reading, and then all threads of the cluster write.  The
// barrier makes in-place calls (kv_lens = lens, free_left = free_count) safe
// without any scratch memory, atomics or order between CTAs.
#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "cache.cuh"
#include "ptx.cuh"

namespace attnprof {
namespace cache {
namespace {

constexpr int kThreads = 1024;
constexpr int kClusterCtas = 8;

struct Counts {
  long long tokens, blocks;
};

// Exclusive prefix of (tokens, blocks) over the CTA's threads, plus `carry`;
// *total becomes carry + the sum over all threads.
__device__ __forceinline__ Counts scan_threads(Counts v, Counts carry, Counts* total,
                                               Counts* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int warps = static_cast<int>(blockDim.x) >> 5;
  Counts in = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long a = __shfl_up_sync(~0u, in.tokens, d), b = __shfl_up_sync(~0u, in.blocks, d);
    if (lane >= d) {
      in.tokens += a;
      in.blocks += b;
    }
  }
  __syncthreads();  // warp_sum of an earlier call has been read
  if (lane == 31) warp_sum[warp] = in;
  __syncthreads();
  if (warp == 0) {
    Counts w = lane < warps ? warp_sum[lane] : Counts{0, 0};
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long a = __shfl_up_sync(~0u, w.tokens, d), b = __shfl_up_sync(~0u, w.blocks, d);
      if (lane >= d) {
        w.tokens += a;
        w.blocks += b;
      }
    }
    if (lane < warps) warp_sum[lane] = w;
  }
  __syncthreads();
  const Counts before = warp > 0 ? warp_sum[warp - 1] : Counts{0, 0};
  const Counts all = warp_sum[warps - 1];
  *total = Counts{carry.tokens + all.tokens, carry.blocks + all.blocks};
  return Counts{carry.tokens + before.tokens + in.tokens - v.tokens,
                carry.blocks + before.blocks + in.blocks - v.blocks};
}

// Largest r with first[r] <= x, for first[0] = 0 <= x (n >= 1 entries).
__device__ __forceinline__ int last_at_most(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Blocks of n >= 0 tokens, up to the largest n: the sum may pass 31 bits.
__device__ __forceinline__ int blocks_of(int n, int shift) {
  return static_cast<int>((static_cast<unsigned>(n) + (1u << shift) - 1) >> shift);
}
__device__ __forceinline__ long long blocks_of(long long n, int shift) {
  return (n + (1 << shift) - 1) >> shift;
}

// Bits 0 and 1 that any thread of the CTA has.
__device__ __forceinline__ int any_of(int bad) {
  if (!__syncthreads_or(bad)) return 0;
  return (__syncthreads_or(bad & 1) ? 1 : 0) | (__syncthreads_or(bad & 2) ? 2 : 0);
}

__device__ __forceinline__ void end_of_reading(int ctas) {
  if (ctas > 1)
    ptx::cluster_sync();
  else
    __syncthreads();
}

struct TablesParams : attn_block_tables_args {
  TablesParams(const attn_block_tables_args& a, int s) : attn_block_tables_args(a), shift(s) {}
  int shift;  // of block_size
};

__global__ void __launch_bounds__(kThreads) tables_kernel(const TablesParams p) {
  extern __shared__ int sm[];
  int* start = sm;                      // [batch] first new token of a request
  int* first = sm + p.batch;            // [batch] rank of its first new block
  int* len = sm + 2 * p.batch;          // [batch] tokens held before
  __shared__ Counts warp_sum[kThreads / 32];
  begin_behind();
  const int count = *p.free_count;
  const int ctas = static_cast<int>(gridDim.x), threads = static_cast<int>(blockDim.x);
  const int mask = (1 << p.shift) - 1;

  Counts total{0, 0};
  int bad = 0;  // bit 0: a row of the table is too short, bit 1: a negative number
  for (int base = 0; base < p.batch; base += threads) {
    const int r = base + static_cast<int>(threadIdx.x);
    Counts v{0, 0};
    int l = 0;
    if (r < p.batch) {
      l = p.lens[r];
      const int n = p.new_lens[r];
      if (l < 0 || n < 0) {
        bad |= 2;
        l = 0;
      } else {
        const long long after = blocks_of(static_cast<long long>(l) + n, p.shift);
        if (after > p.width || static_cast<long long>(l) + n > INT_MAX) bad |= 1;
        v = Counts{n, after - blocks_of(l, p.shift)};
      }
    }
    const Counts at = scan_threads(v, total, &total, warp_sum);
    if (r < p.batch) {  // (kept only where the call is carried out, so that they fit)
      start[r] = static_cast<int>(at.tokens);
      first[r] = static_cast<int>(at.blocks);
      len[r] = l;
    }
  }
  bad = any_of(bad);
  int status = ATTN_BLOCKS_OK;
  if (count < 0 || count > p.num_blocks || total.blocks > count) status = ATTN_BLOCKS_POOL;
  if (bad & 1) status = ATTN_BLOCKS_ROW;
  if (total.tokens > p.tokens) status = ATTN_BLOCKS_SLOTS;
  if (bad & 2) status = ATTN_BLOCKS_NEGATIVE;
  const bool ok = status == ATTN_BLOCKS_OK;
  const int used = ok ? static_cast<int>(total.tokens) : 0;
  const int taken = ok ? static_cast<int>(total.blocks) : 0;

  end_of_reading(ctas);

  const int me = static_cast<int>(blockIdx.x) * threads + static_cast<int>(threadIdx.x);
  const int all = ctas * threads;
  // The step's lengths and the pool's count: one thread each.
  for (int r = me; r < p.batch; r += all) {
    // (p.lens may be p.kv_lens: len[] has it where it is not negative)
    if (ok) {
      const int end = r + 1 < p.batch ? start[r + 1] : used;
      p.kv_lens[r] = len[r] + (end - start[r]);
      p.starts[r] = start[r];
    } else {
      if (p.kv_lens != p.lens) p.kv_lens[r] = p.lens[r];
      p.starts[r] = 0;
    }
  }
  if (me == 0) {
    p.starts[p.batch] = used;
    *p.free_left = count - taken;
    *p.status = status;
  }
  // New blocks into the tables, by the last threads first: the first ones have
  // the slots below, and loads of their own to wait for.
  for (int j = all - 1 - me; j < taken; j += all) {
    const int r = last_at_most(first, p.batch, j);
    const int column = blocks_of(len[r], p.shift) + (j - first[r]);
    p.tables[r * p.table_stride + column] = p.free_blocks[count - 1 - j];
  }
  // Slots, four tokens a thread: one search, then a walk.  A block that the
  // request holds already is read from its table row, a new one from the free
  // list (not from the table, which other threads are writing).
  const bool wide = (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0;
  for (long long t0 = 4ll * me; t0 < p.tokens; t0 += 4ll * all) {
    int out[4] = {-1, -1, -1, -1};
    if (t0 < used) {
      int r = last_at_most(start, p.batch, static_cast<int>(t0));
      int block_rank = -1, id = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = static_cast<int>(t0) + i;
        if (t >= used) break;
        while (r + 1 < p.batch && start[r + 1] <= t) {
          ++r;
          block_rank = -1;
        }
        const int pos = len[r] + (t - start[r]);
        const int b = pos >> p.shift;
        if (b != block_rank) {
          const int held = blocks_of(len[r], p.shift);
          id = b < held ? p.tables[r * p.table_stride + b]
                        : p.free_blocks[count - 1 - (first[r] + b - held)];
          block_rank = b;
        }
        // An id that is not a block of the pool gives no slot.
        if (id >= 0 && id < p.num_blocks) out[i] = (id << p.shift) + (pos & mask);
      }
    }
    if (wide && t0 + 3 < p.tokens) {
      *reinterpret_cast<int4*>(p.slots + t0) = make_int4(out[0], out[1], out[2], out[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t0 + i < p.tokens) p.slots[t0 + i] = out[i];
    }
  }
}

struct TrimParams : attn_block_trim_args {
  TrimParams(const attn_block_trim_args& a, int s) : attn_block_trim_args(a), shift(s) {}
  int shift;
};

__global__ void __launch_bounds__(kThreads) trim_kernel(const TrimParams p) {
  extern __shared__ int sm[];
  int* first = sm;              // [batch] rank of the first block given back
  int* left = sm + p.batch;     // [batch] tokens kept
  __shared__ Counts warp_sum[kThreads / 32];
  begin_behind();
  const int count = *p.free_count;
  const int ctas = static_cast<int>(gridDim.x), threads = static_cast<int>(blockDim.x);

  Counts total{0, 0};
  int bad = 0;
  for (int base = 0; base < p.batch; base += threads) {
    const int r = base + static_cast<int>(threadIdx.x);
    Counts v{0, 0};
    int l = 0;
    if (r < p.batch) {
      l = p.lens[r];
      const int k = p.keep[r];
      if (l < 0 || k < 0) bad |= 2;
      const int held = blocks_of(max(l, 0), p.shift);
      if (held > p.width) bad |= 1;
      l = max(0, min(l, k));
      v.blocks = held - blocks_of(l, p.shift);
    }
    const Counts at = scan_threads(v, total, &total, warp_sum);
    if (r < p.batch) {
      first[r] = static_cast<int>(at.blocks);
      left[r] = l;
    }
  }
  bad = any_of(bad);
  int status = ATTN_BLOCKS_OK;
  // More blocks than the pool has: some were given back before.
  if (count < 0 || count + total.blocks > p.num_blocks) status = ATTN_BLOCKS_POOL;
  if (bad & 1) status = ATTN_BLOCKS_ROW;
  if (bad & 2) status = ATTN_BLOCKS_NEGATIVE;
  const bool ok = status == ATTN_BLOCKS_OK;
  const int back = ok ? static_cast<int>(total.blocks) : 0;

  end_of_reading(ctas);

  const int me = static_cast<int>(blockIdx.x) * threads + static_cast<int>(threadIdx.x);
  const int all = ctas * threads;
  for (int r = me; r < p.batch; r += all) {
    if (ok)
      p.lens_left[r] = left[r];
    else if (p.lens_left != p.lens)
      p.lens_left[r] = p.lens[r];
  }
  if (me == 0) {
    *p.free_left = count + back;
    *p.status = status;
  }
  for (int j = me; j < back; j += all) {
    const int r = last_at_most(first, p.batch, j);
    const int column = blocks_of(left[r], p.shift) + (j - first[r]);
    p.free_blocks[count + j] = p.tables[r * p.table_stride + column];
  }
}

// One CTA where 4 entries a thread do all of the writing, of no more threads
// than that and the requests need (barriers and the scan of fewer warps are
// shorter: 256 requests of a token each 4.1 us with 256 threads, 4.8 with 1024);
// else a cluster.  ints: of shared memory for each request.
template <typename P>
int launch_cluster(void (*kern)(P), const P& p, long long entries, int ints, cudaStream_t st) {
  const int ctas = entries > 4 * kThreads ? kClusterCtas : 1;
  const long long wanted = std::max<long long>((entries + 3) / 4, p.batch);
  const int threads =
      ctas > 1 ? kThreads
               : static_cast<int>(std::min<long long>(std::max(wanted, 1ll) + 31, kThreads)) & ~31;
  const size_t smem = sizeof(int) * ints * p.batch;
  if (smem > 40 * 1024) {  // (the 48 KB of other launches hold the kernel's own too)
    // Once per device and kernel (P names it), for the largest batch: a limit
    // that followed each call's size could be lowered by another thread's.
    static std::atomic<bool> set_up[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ATTN_ERR_CUDA;
    if (dev >= 64 || !set_up[dev].load(std::memory_order_acquire)) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               ints * static_cast<int>(sizeof(int)) * ATTN_BLOCKS_MAX_BATCH) !=
          cudaSuccess)
        return ATTN_ERR_RESOURCE;
      if (dev < 64) set_up[dev].store(true, std::memory_order_release);
    }
  }
  return launch_behind(kern, dim3(static_cast<unsigned>(ctas)), threads, smem, ctas, st, p) ==
                 cudaSuccess
             ? ATTN_OK
             : ATTN_ERR_CUDA;
}

int check_batch(int batch, int width, long long table_stride, int num_blocks, int block_size) {
  if (!block_size_ok(block_size)) return ATTN_ERR_UNSUPPORTED;
  if (batch < 0 || width < 0 || table_stride < width || num_blocks <= 0)
    return ATTN_ERR_INVALID_ARG;
  if (static_cast<long long>(num_blocks) * block_size > INT_MAX) return ATTN_ERR_INVALID_ARG;
  if (batch > ATTN_BLOCKS_MAX_BATCH) return ATTN_ERR_UNSUPPORTED;
  return ATTN_OK;
}

}  // namespace
}  // namespace cache
}  // namespace attnprof

using namespace attnprof::cache;

extern "C" int attn_block_tables(const attn_block_tables_args* args, void* stream) {
  if (!args) return ATTN_ERR_INVALID_ARG;
  const attn_block_tables_args& a = *args;
  const int rc = check_batch(a.batch, a.width, a.table_stride, a.num_blocks, a.block_size);
  if (rc != ATTN_OK) return rc;
  if (a.tokens < 0) return ATTN_ERR_INVALID_ARG;
  if (!a.free_blocks || !a.free_count || !a.starts || !a.free_left || !a.status)
    return ATTN_ERR_INVALID_ARG;
  if (a.batch > 0 && (!a.lens || !a.new_lens || !a.kv_lens)) return ATTN_ERR_INVALID_ARG;
  if ((a.batch > 0 && a.width > 0 && !a.tables) || (a.tokens > 0 && !a.slots))
    return ATTN_ERR_INVALID_ARG;
  for (const void* x : {static_cast<const void*>(a.lens), static_cast<const void*>(a.new_lens),
                        static_cast<const void*>(a.tables), static_cast<const void*>(a.free_blocks),
                        static_cast<const void*>(a.free_count), static_cast<const void*>(a.kv_lens),
                        static_cast<const void*>(a.starts), static_cast<const void*>(a.slots),
                        static_cast<const void*>(a.free_left), static_cast<const void*>(a.status)})
    if (!aligned(x, 4)) return ATTN_ERR_MISALIGNED;
  const TablesParams p{a, shift_of(a.block_size)};
  return launch_cluster(tables_kernel, p, a.tokens, 3, static_cast<cudaStream_t>(stream));
}

extern "C" int attn_block_trim(const attn_block_trim_args* args, void* stream) {
  if (!args) return ATTN_ERR_INVALID_ARG;
  const attn_block_trim_args& a = *args;
  const int rc = check_batch(a.batch, a.width, a.table_stride, a.num_blocks, a.block_size);
  if (rc != ATTN_OK) return rc;
  if (!a.free_blocks || !a.free_count || !a.free_left || !a.status) return ATTN_ERR_INVALID_ARG;
  if (a.batch > 0 && (!a.lens || !a.keep || !a.lens_left)) return ATTN_ERR_INVALID_ARG;
  if (a.batch > 0 && a.width > 0 && !a.tables) return ATTN_ERR_INVALID_ARG;
  for (const void* x : {static_cast<const void*>(a.lens), static_cast<const void*>(a.keep),
                        static_cast<const void*>(a.tables), static_cast<const void*>(a.free_blocks),
                        static_cast<const void*>(a.free_count),
                        static_cast<const void*>(a.lens_left),
                        static_cast<const void*>(a.free_left), static_cast<const void*>(a.status)})
    if (!aligned(x, 4)) return ATTN_ERR_MISALIGNED;
  const TrimParams p{a, shift_of(a.block_size)};
  const long long most = static_cast<long long>(a.batch) * a.width;
  return launch_cluster(trim_kernel, p, std::min<long long>(most, a.num_blocks), 2,
                        static_cast<cudaStream_t>(stream));
}
