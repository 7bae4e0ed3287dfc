// Attention over the 8-bit cache for few query rows a request (single tokens,
// drafts): every key and value is read once from HBM, so the bytes of the
// codes bound it.
//
// Work.  A unit is 8 NT query rows (token x head of the group) of one request
// and kv head, over chunks of 256 keys; all units' chunks, in order, are cut
// into equal ranges, one a CTA, whatever the requests' lengths (a unit counts
// as one chunk more than it has, for what it costs to begin).  A range may
// hold parts of two units and any number of whole ones; whole units are
// written at once, parts go to the workspace as (max, sum, O) and a second
// kernel joins them in the order of the keys, so results do not depend on which
// CTA came first.  The ranges are found by every CTA from the lengths alone.
//
// Inside a CTA one warp fetches and four compute.  The fetching warp walks
// through the CTA's range, over the ends of units, and keeps a ring of steps
// full: per step 128 (D = 128) or 256 keys' codes of K and V by TMA, 16 keys at a time,
// under the 128-byte swizzle, and their blocks' scales by cp.async.  HBM needs
// 6.5 TB/s times some 1.2 us on its way, 53 KB an SM; two CTAs' rings hold 192.
// (Codes read straight into registers by the computing warps: 4.0 TB/s on 64
// requests of 5 to 8191 tokens; a ring for each warp that ran empty at each
// unit's end: 4.7; this form: 5.9, 91 us, 4.8 of them the joining kernel.)
// Each computing warp takes 32 or 64 keys of a step.  S^T = K Q^T and O^T =
// V^T P^T run on m16n8k16 MMAs with the keys (then the head dimension) on the 16
// side and 8 query rows on the other, so that the 1 to 8 rows of a decode step
// waste nothing; tcgen05's smallest tile of 64 to 128 rows would be almost
// empty.  Which key or which head dimension a lane holds is free in a
// contraction as long as both operands agree, so lanes take 16 bytes of a row
// and convert them in place.
// K's scale multiplies the scores in f32; V's scale multiplies each block's
// sum of p v in f32, so no scale is rounded.  P is rounded to f16, by at most
// 2^-11 of itself as an f16 result is (a bf16 result by 2^-8): it is held as
// 2^7 p (p up to 2^8 between two moves of the maximum), so that also weights down
// to 2^-21 of the largest keep all their bits, and smaller ones an absolute
// accuracy of 2^-32 of it.  Maximum, sum and O are f32.
// bf16 queries become f16 times a power of two per row: elements down to 2^-31
// of the row's largest keep all their bits, smaller ones an absolute accuracy of
// 2^-39 of it.
//
// At 17 to 32 rows, D = 64, and 9 to 16 rows, D = 128, O, S, P^T and the words
// of V do not all fit the registers (ptxas: 112 to 262 bytes of spill stores, 216
// to 516 of loads; 8 requests of 4000 tokens: 32 and 24 us, where their bytes
// take 5 and 10).
#include <atomic>
#include <climits>

#include "attn_host.cuh"
#include "cached_attn.cuh"

namespace attnprof {
unsigned long long current_timeout_ns();
int current_fault_mode();

namespace cache {
namespace {

constexpr int kWarps = 4;                    // that compute
constexpr int kThreads = 256;                // two warpgroups: computing, fetching (one warp of it)
constexpr int kChunk = 256;                  // keys
constexpr int kOver = 1;                     // chunks that beginning a unit counts for
// Requests of up to this many chunks are not cut: a second kernel would cost
// more than the keys that it lets other SMs read.  (32 heads over 8, D = 128, in
// graphs: 16 requests of 500 tokens 8.4 us whole, 12.3 cut; 64 of them 17.9 and
// 21.3; 200 46.5 and 46.6.  Of 1000 tokens, 1 request 11.1 and 9.7, 200 74 and 65.)
constexpr int kWholeChunks = 2;
constexpr float kMove = 8.f;                 // growth of the maximum (log2) that moves it
constexpr float kLift = 7.f;                 // P is held as 2^kLift p

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

__device__ __forceinline__ uint32_t byte_perm(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 or 8 bytes of codes (a lane's share of one row) from shared memory.
template <int WORDS>
struct Words {
  uint32_t w[WORDS];
};
template <int WORDS>
__device__ __forceinline__ void load_codes(Words<WORDS>& d, uint32_t a) {
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(d.w[0]), "=r"(d.w[1]), "=r"(d.w[2]), "=r"(d.w[3])
                 : "r"(a)
                 : "memory");
  else
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(d.w[0]), "=r"(d.w[1]) : "r"(a) : "memory");
}

// ---------------------------------------------------------------------------
// The cut of all work into ranges.
// ---------------------------------------------------------------------------
struct Shape {
  int units, chunks, weight;  // of one request: its units, and the chunks and weight of each
  __device__ __forceinline__ long long work() const {
    return static_cast<long long>(units) * weight;
  }
};

template <int NT>
__device__ __forceinline__ Shape shape_of(const CachedParams& p, const Request& r) {
  const long long rows = static_cast<long long>(r.n) * p.group;
  if (rows == 0 || rows > p.rows_most) return Shape{0, 1, 1};
  const int chunks = max(1, (r.kv + kChunk - 1) / kChunk);
  return Shape{p.kv_heads * static_cast<int>((rows + 8 * NT - 1) / (8 * NT)), chunks,
               p.whole ? 1 : chunks + kOver};
}

struct Place {
  int request;
  long long before;  // work of all requests in front of it
};

// x / y for 0 <= x, 0 < y, the quotient in 32 bits; nearly all work counts fit 32
// bits, and a 64-bit division is long.
__device__ __forceinline__ int quotient(long long x, long long y) {
  return ((x | y) >> 32) != 0 ? static_cast<int>(x / y)
                              : static_cast<int>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y));
}

// Sum of all requests' work; a place in it is looked up afterwards: each
// thread keeps the sum of its share of the requests.
template <int NT, bool FROM_L2 = false>
__device__ __forceinline__ long long count_work(const CachedParams& p, long long* part) {
  const int each = (p.batch + blockDim.x - 1) / blockDim.x;
  const int first = static_cast<int>(threadIdx.x) * each;
  long long sum = 0;
  for (int r = first; r < min(first + each, p.batch); ++r) {
    sum += shape_of<NT>(p, request_at<FROM_L2>(p, r)).work();
  }
  // Inclusive prefix over the threads.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long a = __shfl_up_sync(~0u, sum, d);
    if (lane >= d) sum += a;
  }
  __shared__ long long warp_sum[32];
  if (lane == 31) warp_sum[warp] = sum;
  __syncthreads();
  long long before = 0;
  for (int w = 0; w < warp; ++w) before += warp_sum[w];
  part[threadIdx.x] = before + sum;
  __syncthreads();
  return part[blockDim.x - 1];
}

// The request that holds place `at` (below the total); by one thread.
template <int NT, bool FROM_L2 = false>
__device__ __forceinline__ Place find_place(const CachedParams& p, const long long* part,
                                            long long at) {
  int lo = -1, hi = static_cast<int>(blockDim.x) - 1;  // first thread whose prefix is above `at`
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (part[mid] > at) hi = mid; else lo = mid;
  }
  const int each = (p.batch + blockDim.x - 1) / blockDim.x;
  Place pl{hi * each, hi > 0 ? part[hi - 1] : 0};
  while (true) {
    const long long w = shape_of<NT>(p, request_at<FROM_L2>(p, pl.request)).work();
    if (pl.before + w > at || pl.request + 1 >= p.batch) return pl;
    pl.before += w;
    ++pl.request;
  }
}

// The same for up to kLaneRequests requests, by every warp for itself and so
// without a barrier: a lane has up to four requests in a row.
constexpr int kLaneRequests = 128;
struct Lanes {
  long long work, upto;  // of the lane's requests; of all up to and with them
};
template <int NT, bool FROM_L2 = false>
__device__ __forceinline__ Lanes count_lanes(const CachedParams& p, long long* total) {
  const int lane = threadIdx.x & 31, each = (p.batch + 31) / 32;
  Lanes x{0, 0};
  for (int r = lane * each; r < min(lane * each + each, p.batch); ++r)
    x.work += shape_of<NT>(p, request_at<FROM_L2>(p, r)).work();
  x.upto = x.work;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long a = __shfl_up_sync(~0u, x.upto, d);
    if (lane >= d) x.upto += a;
  }
  *total = __shfl_sync(~0u, x.upto, 31);
  return x;
}
template <int NT, bool FROM_L2 = false>
__device__ __forceinline__ Place place_in(const CachedParams& p, const Lanes& x, long long at) {
  const int each = (p.batch + 31) / 32;
  const int lane = __ffs(__ballot_sync(~0u, x.upto > at)) - 1;
  Place pl{lane * each, __shfl_sync(~0u, x.upto - x.work, lane)};
  for (; pl.request + 1 < min(lane * each + each, p.batch); ++pl.request) {
    const long long w = shape_of<NT>(p, request_at<FROM_L2>(p, pl.request)).work();
    if (pl.before + w > at) break;
    pl.before += w;
  }
  return pl;
}

__device__ __forceinline__ long long work_each(long long total, int ctas) {
  return quotient(total + ctas - 1, ctas);
}


// Chunks [c0, c1) of one unit.
struct Part {
  Request rq;
  int request, kvh, row0, c0, c1, chunks;
};

// A CTA's range, part by part.
template <int NT>
struct Cursor {
  long long at, stop;
  Place pl;
  __device__ __forceinline__ bool next(const CachedParams& p, Part& x) {
    while (at < stop && pl.request < p.batch) {
      x.rq = request_at(p, pl.request);
      const Shape sh = shape_of<NT>(p, x.rq);
      if (at >= pl.before + sh.work()) {
        pl.before += sh.work();
        ++pl.request;
        continue;
      }
      const int w = sh.weight;
      const int unit = quotient(at - pl.before, w);
      const int off = static_cast<int>(at - pl.before - static_cast<long long>(unit) * w);
      const int end = static_cast<int>(min(static_cast<long long>(w), off + (stop - at)));
      at += end - off;
      x.c0 = p.whole ? 0 : max(0, off - kOver);
      x.c1 = p.whole ? sh.chunks : max(0, end - kOver);
      if (x.c0 == x.c1) continue;
      const int tiles = sh.units / p.kv_heads;
      x.request = pl.request;
      x.chunks = sh.chunks;
      x.kvh = unit / tiles;
      x.row0 = (unit - x.kvh * tiles) * 8 * NT;
      return true;
    }
    return false;
  }
};

// Parts in the workspace: [rows][D] f32 of O for all slots, then (max, sum)
// per row.  CTA c has slot 2 c + 1 for the part that begins its unit and slot
// 2 c for one that begins inside it (it has at most one of each).
template <int NT, int D>
struct Parts {
  static constexpr int kRows = 8 * NT;
  static __device__ __forceinline__ float* o(float* ws, long long slot) {
    return ws + slot * kRows * D;
  }
  static __device__ __forceinline__ float2* ml(float* ws, long long slots, long long slot) {
    return reinterpret_cast<float2*>(ws + slots * kRows * D) + slot * kRows;
  }
};

// ---------------------------------------------------------------------------
// The kernel.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ uint32_t pack_out(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_out<__half>(float a, float b) { return pack_half2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack_out<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr int kStageBytes = 32768;  // a step's codes of K, then of V

template <int D, int NT>
struct Smem {
  static constexpr int kGroup = 16 * D;                          // bytes of 16 keys
  static constexpr int kGroups = kStageBytes / 2 / kGroup;       // of a step: 8 or 16
  static constexpr int kStages = NT >= 4 ? 2 : 3;
  static constexpr int kOffHop = kStages * kStageBytes;          // a warp's sums on their way
  static constexpr int kHop = 32 * NT * (D / 4 + 4) * 4;
  static constexpr int kOffQ = kOffHop + kHop;                   // Q operands (NT = 4)
  static constexpr int kOffScale = kOffQ + (NT >= 4 ? NT * (D / 16) * 32 * 8 : 0);
  static constexpr int kOffBar = kOffScale + kStages * 2 * kGroups * 4;
  static constexpr int kBytes = kOffBar + 16 * kStages + 1024;   // + alignment
  static_assert(kThreads * 8 <= kHop, "the prefix sums use the hop's place first");
  static_assert(2 * (kBytes + 2048) <= 228 * 1024, "two CTAs an SM");
};

struct SplitParams : CachedParams {
  int* status;
  unsigned long long timeout_ns;
  int fault_mode;  // 1: nothing is fetched (test of the bounded waits)
};

// Named barriers: sums handed from warp h + 1 to warp h, the last reader done,
// Q operands in shared memory.
constexpr int kBarHop = 1, kBarRead = 4, kBarQ = 5;

__device__ __forceinline__ void named_bar_arrive(uint32_t id, uint32_t nthreads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}

// The fetching warp.  Lane i holds the block of group i of 32 (-1: no keys
// there, or no block of the pool) and fetches that group's codes and scales.
template <int D, int NT>
__device__ void fetch_role(const CUtensorMap* map_k, const CUtensorMap* map_v,
                           const SplitParams& p, Cursor<NT> cursor, uint32_t sbase,
                           const WaitCtx& w) {
  using S = Smem<D, NT>;
  constexpr int kPerBatch = 32 / S::kGroups;  // steps whose blocks the lanes hold
  const int lane = threadIdx.x & 31;
  const int mine = lane % S::kGroups;         // group of a step
  const uint32_t full = sbase + S::kOffBar, empty = full + 8 * S::kStages;
  int put = 0, sent = 0;
  uint32_t parity = 1;  // of the place's emptying; at first all are empty
  Part x;
  bool ok = true;
  while (ok && cursor.next(p, x)) {
    const int* table = p.tables + x.request * p.table_stride;
    const int key_end = min(x.c1 * kChunk, x.rq.kv);
    auto block_at = [&](int key) {
      if (key < key_end) {
        const int b = table[key >> p.shift];
        if (b >= 0 && b < p.num_blocks) return b;
      }
      return -1;
    };
    const int begin = x.c0 * kChunk + 16 * lane;
    int id = block_at(begin), id_next = block_at(begin + 512);
    for (int key0 = x.c0 * kChunk; key0 < key_end && ok; key0 += 512) {
#pragma unroll
      for (int s = 0; s < kPerBatch; ++s) {
        if (key0 + s * 16 * S::kGroups >= key_end) break;
        ok = __all_sync(~0u, wait_bar(empty + 8 * put, parity, w, kSiteKvEmpty));
        if (!ok) break;
        const bool turn = lane / S::kGroups == s;
        const bool there = turn && id >= 0;
        const int n = __popc(__ballot_sync(~0u, there));
        const uint32_t bar = full + 8 * put;
        if (lane == 0) ptx::mbar_arrive_expect_tx(bar, n * 2 * S::kGroup);
        __syncwarp();
        const uint32_t scale_at = sbase + S::kOffScale + (put * 2 * S::kGroups + mine) * 4;
        if (there) {
          const int off = (key0 + 16 * lane) & ((1 << p.shift) - 1);
          const int piece = id * p.kv_heads + x.kvh;
          const uint32_t at = sbase + put * kStageBytes + mine * S::kGroup;
          ptx::tma_load_3d(at, map_k, bar, 0, D == 128 ? off : off / 2, piece);
          ptx::tma_load_3d(at + kStageBytes / 2, map_v, bar, 0, D == 128 ? off : off / 2, piece);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(scale_at),
                       "l"(p.ks + piece)
                       : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(scale_at + 4 * S::kGroups),
                       "l"(p.vs + piece)
                       : "memory");
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar)
                       : "memory");
        } else if (turn) {  // a negative scale: nothing here
          ptx::st_shared_f32(scale_at, -1.f);
          ptx::st_shared_f32(scale_at + 4 * S::kGroups, 0.f);
          ptx::mbar_arrive(bar);
        }
        ++sent;
        if (++put == S::kStages) {
          put = 0;
          parity ^= 1;
        }
      }
      id = id_next;
      id_next = block_at(key0 + 1024 + 16 * lane);
    }
  }
  // After a wait that ran out (the host reads of it in the status word): copies
  // on their way end before the shared memory that they go to does.
  if (*w.abort) {
    for (int i = max(0, sent - S::kStages); i < sent; ++i) {
      const unsigned long long t0 = ptx::globaltimer_ns();
      while (!ptx::mbar_try_wait(full + 8 * (i % S::kStages), (i / S::kStages) & 1) &&
             ptx::globaltimer_ns() - t0 < p.timeout_ns) {
      }
    }
  }
}

template <typename T, int CODE, int D, int NT>
__device__ void compute_role(const SplitParams& p, Cursor<NT> cursor, uint32_t sbase,
                             uint8_t* smem, const WaitCtx& w) {
  using S = Smem<D, NT>;
  constexpr int KSTEPS = D / 16;               // MMAs along the head dimension
  constexpr int MT = D / 16;                   // 16-row tiles of O^T
  constexpr int VW = D / 32;                   // words of a V row that a lane holds (D / 8 bytes)
  constexpr int KP = D / 64;                   // 16-byte pieces of a K row that a lane holds
  constexpr bool kQShared = NT >= 4;           // Q operands from shared memory, to save registers
  constexpr int KT = S::kGroups / kWarps;      // 16-key tiles of a warp's step: 2 or 4
  constexpr int kStep = 16 * S::kGroups;       // keys of a step
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t full = sbase + S::kOffBar, empty = full + 8 * S::kStages;
  uint2* q_sh = reinterpret_cast<uint2*>(smem + S::kOffQ);
  float* hop = reinterpret_cast<float*>(smem + S::kOffHop) + lane;

  // Where the lane's pieces lie in a group's 16 rows (D = 64: 8 rows of two
  // keys) under the 128-byte swizzle: 16-byte piece c of row r at c ^ (r % 8).
  uint32_t k_at[2][KP], v_at[4];
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int pc = 0; pc < KP; ++pc) {
      const int key = g + 8 * r;
      k_at[r][pc] = D == 128 ? key * 128 + (((4 * pc + t) ^ (key & 7)) << 4)
                             : (key >> 1) * 128 + ((((key & 1) * 4 + t) ^ (key >> 1)) << 4);
    }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int key = 2 * t + (r & 1) + 8 * (r >> 1);
    v_at[r] = D == 128 ? key * 128 + ((g ^ (key & 7)) << 4)
                       : (key >> 1) * 128 + ((((key & 1) * 4 + (g >> 1)) ^ (key >> 1)) << 4) +
                             8 * (g & 1);
  }

  int take = 0;
  uint32_t parity = 0;
  bool ok = true, first = true;
  Part x;
  while (cursor.next(p, x)) {
    const Request& rq = x.rq;
    const int rows_in = rq.n * p.group;
    if constexpr (kQShared) ptx::named_bar_sync(kBarQ, 32 * kWarps);  // the last ones are used up
    // Q operands: lane (g, t) holds row 8 nt + g, the head dimensions that its
    // K bytes belong to.
    uint32_t qb[kQShared ? 1 : NT][kQShared ? 1 : KSTEPS][2];
    float row_f[NT][2];  // score factor of rows 2t, 2t + 1
    int limit[NT][2];    // keys that they see
    int least = INT_MAX;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = x.row0 + 8 * nt + g;
      const bool live = row < rows_in;
      const int tok = live ? row / p.group : 0;
      const T* qr = static_cast<const T*>(p.q) + (rq.start + tok) * p.q_token +
                    (x.kvh * p.group + (live ? row - tok * p.group : 0)) * p.q_head;
      float f = 1.f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        uint32_t top = 0;
#pragma unroll
        for (int pc = 0; pc < KP; ++pc)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 w = live ? *reinterpret_cast<const uint4*>(qr + 64 * pc + 16 * t + 8 * j)
                                 : make_uint4(0, 0, 0, 0);
            top = __vmaxu2(top, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu),
                                         __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
          }
        top = max(top & 0xffffu, top >> 16);
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        // The row's largest |q| to [2^14, 2^15); rows that are zero or not
        // finite as they are.
        const int e = static_cast<int>(top >> 7) - 127;
        if (top > 0 && e < 128) f = power_of_two(max(e - 14, -112));
      }
      const float inv = 1.f / f;  // a power of two
      const float mine = f * p.scale_log2;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const int d = 64 * (ks / 4) + 16 * t + 4 * (ks % 4);
        uint2 b = make_uint2(0, 0);
        if (live) {
          if constexpr (std::is_same<T, __half>::value) {
            b = *reinterpret_cast<const uint2*>(qr + d);
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(qr + d);
            b.x = pack_half2(__uint_as_float(v.x << 16) * inv,
                             __uint_as_float(v.x & 0xffff0000u) * inv);
            b.y = pack_half2(__uint_as_float(v.y << 16) * inv,
                             __uint_as_float(v.y & 0xffff0000u) * inv);
          }
        }
        if constexpr (kQShared) {
          if (warp == 0) q_sh[(nt * KSTEPS + ks) * 32 + lane] = b;
        } else {
          qb[nt][ks][0] = b.x;
          qb[nt][ks][1] = b.y;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        row_f[nt][j] = __shfl_sync(~0u, mine, (2 * t + j) * 4);
        const int r = x.row0 + 8 * nt + 2 * t + j;
        // (rows behind the last one: zeros that see everything)
        limit[nt][j] = r < rows_in && p.causal ? rq.before + r / p.group + 1 : rq.kv;
        limit[nt][j] = min(limit[nt][j], rq.kv);
        least = min(least, limit[nt][j]);
      }
    }
    least = __reduce_min_sync(~0u, least);
    if constexpr (kQShared) ptx::named_bar_sync(kBarQ, 32 * kWarps);

    float o[NT][MT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    const int key_end = min(x.c1 * kChunk, rq.kv);
    for (int key_s = x.c0 * kChunk; key_s < key_end; key_s += kStep) {
      const int key0 = key_s + 16 * KT * warp;
      const uint32_t from = sbase + take * kStageBytes + warp * KT * S::kGroup;
      const float* scale = reinterpret_cast<const float*>(smem + S::kOffScale) +
                           take * 2 * S::kGroups + warp * KT;
      // (After a wait that ran out this goes on without waiting, so that all
      // warps meet at their barriers; the status word tells the host.)
      if (ok) ok = __all_sync(~0u, wait_bar(full + 8 * take, parity, w, kSiteKvFull));
      // S^T = K Q^T
      float sc[NT][KT][4];
      float kscale[KT], vsc[KT];
      bool held[KT];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        kscale[k] = scale[k];
        vsc[k] = scale[S::kGroups + k];
        held[k] = !(kscale[k] < 0.f);
        if (!held[k]) kscale[k] = 1.f;  // (of scores that will be -inf)
        Words<4> kw[2][KP];  // [row g, row g + 8][piece]
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int pc = 0; pc < KP; ++pc) load_codes(kw[r][pc], from + k * S::kGroup + k_at[r][pc]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][k][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
          const uint32_t w0 = kw[0][ks / 4].w[ks % 4], w1 = kw[1][ks / 4].w[ks % 4];
          const uint32_t a[4] = {Code<CODE>::half2_lo(w0), Code<CODE>::half2_lo(w1),
                                 Code<CODE>::half2_hi(w0), Code<CODE>::half2_hi(w1)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if constexpr (kQShared) {
              const uint2 b = q_sh[(nt * KSTEPS + ks) * 32 + lane];
              mma_16816(sc[nt][k], a, b.x, b.y);
            } else {
              mma_16816(sc[nt][k], a, qb[nt][ks][0], qb[nt][ks][1]);
            }
          }
        }
      }

      // Masks, where not every key is there for every row.
      bool clean = key0 + 16 * KT <= least;
#pragma unroll
      for (int k = 0; k < KT; ++k) clean &= held[k];
      if (!clean) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!held[k] || key0 + 16 * k + 8 * (i >> 1) + g >= limit[nt][i & 1])
                sc[nt][k][i] = -INFINITY;
      }
      // The maximum moves only when a score exceeds it by 2^kMove (as the first
      // ones do): then, and only then, the lanes of a row agree on it and the
      // sums are rescaled.
      float top[NT][2];
      bool move = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = -INFINITY;
#pragma unroll
          for (int k = 0; k < KT; ++k)
            x = fmaxf(x, fmaxf(sc[nt][k][j], sc[nt][k][2 + j]) * (kscale[k] * row_f[nt][j]));
          top[nt][j] = x;
          move |= x > m[nt][j] + kMove;
        }
      if (__any_sync(~0u, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float x = top[nt][j];
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
            const float now = fmaxf(m[nt][j], x);
            const float alpha = now == -INFINITY ? 1.f : ptx::ex2_approx(m[nt][j] - now);
            m[nt][j] = now;
            l[nt][j] *= alpha;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              o[nt][mt][j] *= alpha;
              o[nt][mt][2 + j] *= alpha;
            }
          }
      }
      // P.  (A masked score is -inf; times a factor that is NaN or 0 it is not.)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float neg = m[nt][j] == -INFINITY ? 0.f : kLift - m[nt][j];
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            const float f = kscale[k] * row_f[nt][j];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x = sc[nt][k][2 * h + j];
              float e = ptx::ex2_approx(fmaf(x, f, neg));
              if (!clean && x == -INFINITY) e = 0.f;
              sc[nt][k][2 * h + j] = e;
              sum += e;
            }
          }
          l[nt][j] += sum;
        }

      // P^T as the second operand: keys move from lanes' rows to their columns.
      uint32_t pb[NT][KT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          pb[nt][k][0] = transpose_8x8(pack_half2(sc[nt][k][0], sc[nt][k][1]));
          pb[nt][k][1] = transpose_8x8(pack_half2(sc[nt][k][2], sc[nt][k][3]));
        }
      // V: [tile][keys 2t, 2t + 1, 2t + 8, 2t + 9].
      Words<VW> vw[KT][4];
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          load_codes(vw[k][r], from + kStageBytes / 2 + k * S::kGroup + v_at[r]);
      if (!clean) {
        // What lies behind the last token, or where nothing was fetched, may be
        // any bits: 0 * NaN would reach a sum.
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!held[k] || key0 + 16 * k + 2 * t + (r & 1) + 8 * (r >> 1) >= rq.kv) {
#pragma unroll
              for (int i = 0; i < VW; ++i) vw[k][r].w[i] = 0u;
            }
      }
      __syncwarp();  // every lane has its codes: the place may be filled again
      if (lane == 0) ptx::mbar_arrive(empty + 8 * take);
      if (++take == S::kStages) {
        take = 0;
        parity ^= 1;
      }
      // O^T += scale (V^T P^T), the scale once a block: tiles of one block add
      // up first (their scale is the first one's: others may have no token).
      const int joint = p.shift > 5 ? KT : p.shift > 4 ? 2 : 1;
#pragma unroll
      for (int mp = 0; mp < MT / 2; ++mp) {
        float acc[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[h][nt][i] = 0.f;
        float f = 0.f;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const uint32_t x0 = byte_perm(vw[k][0].w[mp], vw[k][1].w[mp], 0x5140);
          const uint32_t x1 = byte_perm(vw[k][0].w[mp], vw[k][1].w[mp], 0x7362);
          const uint32_t y0 = byte_perm(vw[k][2].w[mp], vw[k][3].w[mp], 0x5140);
          const uint32_t y1 = byte_perm(vw[k][2].w[mp], vw[k][3].w[mp], 0x7362);
          const uint32_t a0[4] = {Code<CODE>::half2_lo(x0), Code<CODE>::half2_hi(x0),
                                  Code<CODE>::half2_lo(y0), Code<CODE>::half2_hi(y0)};
          const uint32_t a1[4] = {Code<CODE>::half2_lo(x1), Code<CODE>::half2_hi(x1),
                                  Code<CODE>::half2_lo(y1), Code<CODE>::half2_hi(y1)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_16816(acc[0][nt], a0, pb[nt][k][0], pb[nt][k][1]);
            mma_16816(acc[1][nt], a1, pb[nt][k][0], pb[nt][k][1]);
          }
          if ((k & (joint - 1)) == 0) f = vsc[k];
          if (((k + 1) & (joint - 1)) == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  o[nt][2 * mp + h][i] = fmaf(acc[h][nt][i], f, o[nt][2 * mp + h][i]);
                  acc[h][nt][i] = 0.f;
                }
          }
        }
      }
    }

    // The four warps' sums together, from warp 3 to warp 0, lane by lane (the
    // same lane of each warp holds the same rows and head dimensions).
    if (warp == kWarps - 1) {
      if (!first) ptx::named_bar_sync(kBarRead, 64);  // by warp 0, in the unit before
    } else {
      ptx::named_bar_sync(kBarHop + warp, 64);
      float* from = hop;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mine[2], other[2];
#pragma unroll
        for (int j = 0; j < 2; ++j, from += 64) {
          const float m2 = from[0], l2 = from[32];
          const float now = fmaxf(m[nt][j], m2), base = now == -INFINITY ? 0.f : now;
          mine[j] = ptx::ex2_approx(m[nt][j] - base);
          other[j] = ptx::ex2_approx(m2 - base);
          m[nt][j] = now;
          l[nt][j] = l[nt][j] * mine[j] + l2 * other[j];
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i, from += 32)
            o[nt][mt][i] = o[nt][mt][i] * mine[i & 1] + *from * other[i & 1];
      }
    }
    first = false;
    if (warp > 0) {
      float* to = hop;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 2; ++j, to += 64) {
          to[0] = m[nt][j];
          to[32] = l[nt][j];
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i, to += 32) *to = o[nt][mt][i];
      }
      named_bar_arrive(kBarHop + warp - 1, 64);
      continue;
    }
    named_bar_arrive(kBarRead, 64);
    const bool all_keys = x.c0 == 0 && x.c1 == x.chunks;
    const long long slot = 2ll * blockIdx.x + (x.c0 == 0 ? 1 : 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[nt][j];
        sum += __shfl_xor_sync(~0u, sum, 4);
        sum += __shfl_xor_sync(~0u, sum, 8);
        sum += __shfl_xor_sync(~0u, sum, 16);
        const int r = 8 * nt + 2 * t + j, row = x.row0 + r;
        if (row >= rows_in) continue;
        if (all_keys) {
          const float n = m[nt][j] == -INFINITY && sum == sum ? 0.f : 1.f / sum;
          const int tok = row / p.group;
          uint4* dst = reinterpret_cast<uint4*>(
              static_cast<T*>(p.out) + (rq.start + tok) * p.o_token +
              (x.kvh * p.group + row - tok * p.group) * p.o_head + 4 * VW * g);
#pragma unroll
          for (int mt = 0; mt < MT; mt += 4)
            dst[mt / 4] = make_uint4(pack_out<T>(o[nt][mt][j] * n, o[nt][mt][2 + j] * n),
                                     pack_out<T>(o[nt][mt + 1][j] * n, o[nt][mt + 1][2 + j] * n),
                                     pack_out<T>(o[nt][mt + 2][j] * n, o[nt][mt + 2][2 + j] * n),
                                     pack_out<T>(o[nt][mt + 3][j] * n, o[nt][mt + 3][2 + j] * n));
        } else {
          float4* dst = reinterpret_cast<float4*>(Parts<NT, D>::o(p.ws, slot) + r * D + 4 * VW * g);
#pragma unroll
          for (int mt = 0; mt < MT; mt += 2)
            dst[mt / 2] = make_float4(o[nt][mt][j], o[nt][mt][2 + j], o[nt][mt + 1][j],
                                      o[nt][mt + 1][2 + j]);
          if (g == 0)
            Parts<NT, D>::ml(p.ws, 2ll * gridDim.x, slot)[r] = make_float2(m[nt][j], sum);
        }
      }
  }
  if (warp == kWarps - 1 && !first) ptx::named_bar_sync(kBarRead, 64);
}

template <typename T, int CODE, int D, int NT>
__global__ void __launch_bounds__(kThreads, 2)
split_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
             const SplitParams p) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL)
  using S = Smem<D, NT>;
  __shared__ Place place;
  __shared__ int abort_flag;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - raw);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      ptx::mbar_init(sbase + S::kOffBar + 8 * i, S::kGroups + 1);
      ptx::mbar_init(sbase + S::kOffBar + 8 * (S::kStages + i), kWarps);
    }
    abort_flag = 0;
    ptx::fence_mbar_init();
  }
  begin_behind();  // only then: the joining kernel reads lengths before it waits
  Cursor<NT> cursor;
  long long total;
  if (p.batch <= kLaneRequests) {
    const Lanes lanes = count_lanes<NT>(p, &total);
    const long long each = work_each(total, gridDim.x);
    cursor.at = each * blockIdx.x;
    cursor.stop = min(cursor.at + each, total);
    if (cursor.at >= cursor.stop) return;
    cursor.pl = place_in<NT>(p, lanes, cursor.at);
    __syncthreads();  // the barriers are there
  } else {
    long long* part_sum = reinterpret_cast<long long*>(smem + S::kOffHop);
    total = count_work<NT>(p, part_sum);
    const long long each = work_each(total, gridDim.x);
    cursor.at = each * blockIdx.x;
    cursor.stop = min(cursor.at + each, total);
    if (cursor.at >= cursor.stop) return;
    if (threadIdx.x == 0) place = find_place<NT>(p, part_sum, cursor.at);
    __syncthreads();
    cursor.pl = place;
  }
  const WaitCtx w{&abort_flag, p.status, p.timeout_ns};
  // Registers: 128 x (216 + 40) = 256 x 128.
  if (warp < kWarps) {
    ptx::setmaxnreg_inc<216>();
    compute_role<T, CODE, D, NT>(p, cursor, sbase, smem, w);
  } else {
    ptx::setmaxnreg_dec<40>();
    if (warp == kWarps && p.fault_mode == 0)
      fetch_role<D, NT>(&map_k, &map_v, p, cursor, sbase, w);
  }
#endif
}

// Parts of one row joined one after the other: a lane has N head dimensions.
template <int N>
struct Sums {
  float top = -INFINITY, sum = 0.f, x[N] = {};
  __device__ __forceinline__ void add(float2 ml, const float* o) {
    float y[N];
    if constexpr (N == 4) {
      const float4 v = *reinterpret_cast<const float4*>(o);
      y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(o);
      y[0] = v.x; y[1] = v.y;
    }
    const float now = fmaxf(top, ml.x), base = now == -INFINITY ? 0.f : now;
    const float a = ptx::ex2_approx(top - base), b = ptx::ex2_approx(ml.x - base);
    top = now;
    sum = sum * a + ml.y * b;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = x[j] * a + y[j] * b;
  }
};

// Joins the parts of the units that were cut.  CTA c > 0 looks at the cut in
// front of range c and, if that is the first cut in its unit, joins the unit:
// the part that ends range c - 1, then those that begin ranges c, c + 1, ...
// One warp a row.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(256) join_kernel(const CachedParams p) {
  constexpr int kRows = 8 * NT;
  __shared__ long long part_sum[256];
  __shared__ Place place;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long total, each, cut;
  Place pl{0, 0};
  if (p.batch <= kLaneRequests) {
    const Lanes lanes = count_lanes<NT, true>(p, &total);
    each = work_each(total, gridDim.x);
    cut = each * (blockIdx.x + 1ll);
    if (cut < total) pl = place_in<NT, true>(p, lanes, cut);
  } else {
    total = count_work<NT, true>(p, part_sum);
    each = work_each(total, gridDim.x);
    cut = each * (blockIdx.x + 1ll);
    if (threadIdx.x == 0 && cut < total) place = find_place<NT, true>(p, part_sum, cut);
    __syncthreads();
    pl = place;
  }
  // By every CTA, those without work too: this kernel may not end before the
  // one in front of it.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (cut >= total) return;
  const Request rq = request_at(p, pl.request);
  const Shape sh = shape_of<NT>(p, rq);
  const int unit = quotient(cut - pl.before, sh.weight);
  const long long begin = pl.before + static_cast<long long>(unit) * sh.weight;
  const long long end = begin + sh.weight;
  // Only if chunks lie in front of this cut, and none in front of the last one.
  if (cut <= begin + kOver || cut - each > begin + kOver) return;
  const int tiles = sh.units / p.kv_heads;
  const int kvh = unit / tiles;
  const int row0 = (unit - kvh * tiles) * kRows;
  const int rows_in = rq.n * p.group;
  const int parts = quotient(end - cut + each - 1, each) + 1;
  const long long slots = 2ll * gridDim.x;

  auto slot_of = [&](int i) { return i == 0 ? 2ll * blockIdx.x + 1 : 2ll * (blockIdx.x + i); };
  constexpr int kPer = D / 32;
  for (int r = warp; r < kRows && row0 + r < rows_in; r += 8) {
    Sums<kPer> s;
#pragma unroll 2
    for (int i = 0; i < parts; ++i)
      s.add(Parts<NT, D>::ml(p.ws, slots, slot_of(i))[r],
            Parts<NT, D>::o(p.ws, slot_of(i)) + r * D + lane * kPer);
    const float n = s.top == -INFINITY && s.sum == s.sum ? 0.f : 1.f / s.sum;
    const int row = row0 + r, tok = row / p.group;
    T* dst = static_cast<T*>(p.out) + (rq.start + tok) * p.o_token +
             (kvh * p.group + row - tok * p.group) * p.o_head + lane * kPer;
    if constexpr (D == 128)
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack_out<T>(s.x[0] * n, s.x[1] * n), pack_out<T>(s.x[2] * n, s.x[3] * n));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack_out<T>(s.x[0] * n, s.x[1] * n);
  }
}

// The same where units are few (at most kFewUnits of at most 32 requests) and
// so have many parts each: a CTA per unit and row, its warps share the parts.
constexpr int kFewUnits = 64;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(256) join_few_kernel(const CachedParams p, int ctas) {
  __shared__ float top_of[8], sum_of[8];
  __shared__ float x_of[8][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Lane r has request r.
  Shape sh{0, 1, 1};
  if (lane < p.batch) sh = shape_of<NT>(p, request_at<true>(p, lane));
  long long total;
  const Lanes lanes = count_lanes<NT, true>(p, &total);
  const long long each = work_each(total, ctas);
  // The request that holds this unit.
  int upto = sh.units;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(~0u, upto, d);
    if (lane >= d) upto += a;
  }
  const int r = __ffs(__ballot_sync(~0u, upto > static_cast<int>(blockIdx.x))) - 1;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (r < 0) return;
  const int units = __shfl_sync(~0u, sh.units, r), weight = __shfl_sync(~0u, sh.weight, r);
  const int unit = static_cast<int>(blockIdx.x) - (__shfl_sync(~0u, upto, r) - units);
  const long long begin = __shfl_sync(~0u, lanes.upto, r) -
                          static_cast<long long>(units - unit) * weight;
  const long long end = begin + weight;
  // Ranges with chunks of the unit: the one that its first chunk lies in, to the last.
  const int c0 = quotient(begin + kOver, each), c1 = quotient(end - 1, each);
  if (c0 == c1) return;  // not cut
  const Request rq = request_at(p, r);
  const int tiles = units / p.kv_heads;
  const int kvh = unit / tiles;
  const int row_in = blockIdx.y, row = (unit - kvh * tiles) * 8 * NT + row_in;
  if (row >= rq.n * p.group) return;
  const long long slots = 2ll * ctas;
  auto slot_of = [&](int c) { return 2ll * c + (c == c0 ? 1 : 0); };

  constexpr int kPer = D / 32;
  Sums<kPer> s;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += 8)
    s.add(Parts<NT, D>::ml(p.ws, slots, slot_of(c))[row_in],
          Parts<NT, D>::o(p.ws, slot_of(c)) + row_in * D + lane * kPer);
  if (lane == 0) {
    top_of[warp] = s.top;
    sum_of[warp] = s.sum;
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) x_of[warp][lane * kPer + j] = s.x[j];
  __syncthreads();
  const int d = 2 * threadIdx.x;  // two head dimensions a thread
  if (d >= D) return;
  float top = top_of[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, top_of[i]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = ptx::ex2_approx(top_of[i] - base);
    sum = fmaf(sum_of[i], f, sum);
    x0 = fmaf(x_of[i][d], f, x0);
    x1 = fmaf(x_of[i][d + 1], f, x1);
  }
  const float n = top == -INFINITY && sum == sum ? 0.f : 1.f / sum;
  const int tok = row / p.group;
  T* dst = static_cast<T*>(p.out) + (rq.start + tok) * p.o_token +
           (kvh * p.group + row - tok * p.group) * p.o_head + d;
  *reinterpret_cast<uint32_t*>(dst) = pack_out<T>(x0 * n, x1 * n);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Rows of 8 that a unit holds: as many as the longest request's rows need;
// where longer requests go to the tiled kernel, what single tokens need.
int row_tiles(int group, int D, int max_new) {
  const long long rows = static_cast<long long>(group) * max_new;
  const long long want = rows <= (D == 64 ? 32 : 16) ? rows : group;
  return want <= 8 ? 1 : want <= 16 || D == 128 ? 2 : 4;
}

constexpr int kMostCtasPerSm = 2;  // by shared memory and registers; bounds the workspace

template <typename T, int CODE, int D, int NT>
int resident_ctas(int* ctas) {
  static std::atomic<int> known[64];  // per device, 0 until it is set up
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ATTN_ERR_CUDA;
  int n = dev < 64 ? known[dev].load(std::memory_order_acquire) : 0;
  if (n == 0) {
    constexpr int smem = Smem<D, NT>::kBytes;
    auto kern = split_kernel<T, CODE, D, NT>;
    int sms = 0, occ = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return ATTN_ERR_RESOURCE;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kThreads, smem) != cudaSuccess)
      return ATTN_ERR_CUDA;
    if (occ < 1) return ATTN_ERR_RESOURCE;
    n = sms * (occ < kMostCtasPerSm ? occ : kMostCtasPerSm);
    if (dev < 64) known[dev].store(n, std::memory_order_release);
  }
  *ctas = n;
  return ATTN_OK;
}

size_t part_bytes(int D, int nt) { return sizeof(float) * 8 * nt * (D + 2) * 2; }

template <typename T, int CODE, int D, int NT>
int launch(const CachedParams& cp, int max_new, void* ws, unsigned long long ws_bytes,
           cudaStream_t st) {
  SplitParams p;
  static_cast<CachedParams&>(p) = cp;
  p.status = device_status_ptr();
  if (p.status == nullptr) return ATTN_ERR_CUDA;
  p.timeout_ns = current_timeout_ns();
  p.fault_mode = current_fault_mode();
  CUtensorMap map_k, map_v;
  if (const int e = codes_map(&map_k, p.kc, p, D)) return e;
  if (const int e = codes_map(&map_v, p.vc, p, D)) return e;
  int ctas = 0;
  const int rc = resident_ctas<T, CODE, D, NT>(&ctas);
  if (rc != ATTN_OK) return rc;
  const long long rows = static_cast<long long>(p.group) * max_new;
  const double units = static_cast<double>(p.batch) * p.kv_heads * ((rows + 8 * NT - 1) / (8 * NT));
  const int chunks = p.capacity <= kChunk ? 1 : (p.capacity + kChunk - 1) / kChunk;
  p.whole = p.capacity <= kWholeChunks * kChunk;
  // No more ranges than there can be chunks.
  const double most = units * (p.whole ? 1 : chunks);
  if (most < ctas) ctas = static_cast<int>(most);
  if (!p.whole && (ws == nullptr || ws_bytes < part_bytes(D, NT) * ctas))
    return ATTN_ERR_WORKSPACE;
  p.ws = static_cast<float*>(ws);
  if (launch_behind(split_kernel<T, CODE, D, NT>, dim3(static_cast<unsigned>(ctas)), kThreads,
                    Smem<D, NT>::kBytes, 0, st, map_k, map_v, p) != cudaSuccess)
    return ATTN_ERR_CUDA;
  if (p.whole || ctas == 1) return ATTN_OK;
  // The joining kernel starts while the first still runs (its search of the
  // cuts overlaps) and waits for it before it reads the parts.
  const bool few = p.batch <= 32 && units <= kFewUnits;
  const CachedParams& base = p;
  const cudaError_t e =
      few ? launch_behind(join_few_kernel<T, D, NT>, dim3(static_cast<unsigned>(units), 8 * NT),
                          256, 0, 0, st, base, ctas)
          : launch_behind(join_kernel<T, D, NT>, dim3(static_cast<unsigned>(ctas)), 256, 0, 0, st,
                          base);
  return e == cudaSuccess ? ATTN_OK : ATTN_ERR_CUDA;
}

template <typename T, int CODE, int D>
int launch_nt(const CachedParams& p, int max_new, void* ws, unsigned long long b, cudaStream_t st) {
  switch (row_tiles(p.group, D, max_new)) {
    case 1: return launch<T, CODE, D, 1>(p, max_new, ws, b, st);
    case 2: return launch<T, CODE, D, 2>(p, max_new, ws, b, st);
    default:
      if constexpr (D == 64) return launch<T, CODE, D, 4>(p, max_new, ws, b, st);
      return ATTN_ERR_UNSUPPORTED;  // (not reached: D = 128 has at most 16 rows here)
  }
}

template <typename T, int CODE>
int launch_d(const CachedParams& p, int D, int n, void* ws, unsigned long long b, cudaStream_t st) {
  return D == 64 ? launch_nt<T, CODE, 64>(p, n, ws, b, st) : launch_nt<T, CODE, 128>(p, n, ws, b, st);
}

template <typename T>
int launch_code(const CachedParams& p, int D, int code, int n, void* ws, unsigned long long b,
                cudaStream_t st) {
  return code == ATTN_CODE_E4M3 ? launch_d<T, ATTN_CODE_E4M3>(p, D, n, ws, b, st)
                                : launch_d<T, ATTN_CODE_INT8>(p, D, n, ws, b, st);
}

}  // namespace

// The codes of a pool as [num_blocks * kv_heads][bytes of a block / 128][128
// bytes], fetched 16 keys at a time with the 128-byte swizzle.
int codes_map(CUtensorMap* m, const void* codes, const CachedParams& p, int D) {
  const EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return ATTN_ERR_CUDA;
  const long long pieces = static_cast<long long>(p.num_blocks) * p.kv_heads;
  if (pieces > INT_MAX) return ATTN_ERR_INVALID_ARG;  // (a coordinate)
  const cuuint64_t block = static_cast<cuuint64_t>(D) << p.shift;
  const cuuint64_t dims[3] = {128, block / 128, static_cast<cuuint64_t>(pieces)};
  const cuuint64_t strides[2] = {128, block};
  const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(16 * D / 128), 1};
  const cuuint32_t one[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? ATTN_OK
             : ATTN_ERR_TENSOR_MAP;
}

int launch_split(const CachedParams& p, int D, int dtype, int code, int max_new, void* ws,
                 unsigned long long ws_bytes, cudaStream_t st) {
  return dtype == ATTN_DTYPE_F16 ? launch_code<__half>(p, D, code, max_new, ws, ws_bytes, st)
                                 : launch_code<__nv_bfloat16>(p, D, code, max_new, ws, ws_bytes, st);
}

int split_workspace(int group, int D, int max_new, int capacity, unsigned long long* bytes) {
  *bytes = 0;
  if (capacity <= kWholeChunks * kChunk) return ATTN_OK;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return ATTN_ERR_CUDA;
  *bytes = part_bytes(D, row_tiles(group, D, max_new)) * sms * kMostCtasPerSm;
  return ATTN_OK;
}

}  // namespace cache
}  // namespace attnprof
