// Attention over the 8-bit cache for many query rows a request (prompts and
// chunks of them): the tensor cores' rate bounds it, 4 D operations a visible
// (row, key).
//
// One CTA takes 256 query rows (token x head of the group, so grouped heads
// share every key and value) of one request and kv head: two tiles of 128 rows
// whose softmax steps take turns, as in the dense kernel of this library.  Per
// 128 keys:
//   * one warp fetches codes by TMA and scales by cp.async (through L2: the row
//     tiles of a head follow each other);
//   * a warpgroup turns them into f16 and writes them into a ring of shared
//     memory tiles in the tensor cores' 128-byte swizzle: 8 bits to 16 once for
//     256 rows.  (Codes read by that warpgroup itself into registers: 1295 us
//     where this form took 988 on 3 chunks of up to 2048 tokens, 32 heads of
//     128 over 8, up to 16,000 keys.)
//   * one thread issues tcgen05.mma: S = Q K^T and O += P V, sums in tensor
//     memory, P read from there too.  At D = 128 its 512 columns hold S and O of
//     both tiles and P overwrites S.  At D = 64 P has columns of its own, a
//     tile's next S is computed during its softmax step, and each tile has a
//     thread of its own, since one thread would hold one tile's S back until it
//     has P of the other (waits of the softmax 1100 -> 240 of 3600 cycles a step);
//   * a warpgroup per tile runs the online softmax, a thread a row, and moves O
//     to a new maximum only when that grew by more than 2^8.
// Now 784 us for those chunks, 1140 TFLOP/s: at D = 128 a step of 128 keys takes
// some 3650 cycles, of which the MMAs 2048, the exponentials 2048 and shared
// memory 2560, and a tile's softmax waits for its P V and next S behind the
// other tile's.  At D = 64 it takes 3500, the softmax warps' own.
//
// Scales.  K's multiplies the scores in f32, 16 keys at a time (no block is
// smaller).  V's must act before the sum over keys: V is held as code * s / r
// * 2^7 (int8: 2^8) in f16, r being the largest V scale of the blocks that the
// unit sees, found first.  For powers of two that is exact down to s = 2^-22 r
// (code and factor only meet f16's end below), and below it the rounding, by
// half of f16's least step, is 2^-32 r at most (the product is formed in f32
// where f16 would not hold the factor); other scales round V to f16 once.  P is rounded to f16 as in the split kernel, held as 2^7 p with p
// up to 2^8 between two moves of the maximum.  bf16 queries become f16 times
// a power of two per row.
#include <atomic>

#include "attn_kernel.cuh"
#include "cached_attn.cuh"

namespace attnprof {
int* device_status_ptr();
unsigned long long current_timeout_ns();
int current_fault_mode();

namespace cache {
namespace {

constexpr int kBM = 128;                 // rows of a tile
constexpr int kBN = 128;                 // keys of a step
constexpr int kUnit = 2 * kBM;           // rows of a CTA
constexpr int kThreads = 512;            // 2 softmax warpgroups, 1 converting, 1 with the issuer
constexpr int kScaleRing = 8;            // steps whose K scales are kept (see fetch_role)
constexpr float kMove = 8.f;             // growth of the maximum (log2) that moves O
constexpr float kLift = 7.f;             // P is held as 2^kLift p

template <int D>
struct Tile {
  static constexpr int kBytes = kBN * D * 2;        // one tile in 16 bits
  static constexpr int kBlock = kBN * 128;          // its 64-column blocks
  static constexpr int kSlots = D == 128 ? 4 : 6;   // of the ring of tiles in 16 bits
  static constexpr int kCodes = kBN * D;            // one tile in 8 bits
  static constexpr int kGroup = 16 * D;             // 16 keys of it
  static constexpr int kStages = D == 128 ? 2 : 4;  // of the ring of tiles in 8 bits
  // Units of 128 rows read each key for fewer rows, and more often from HBM: at
  // D = 128 the second Q tile's place, which they do not need, makes two more.
  static constexpr int kDualStages = 4;
  // Tensor memory columns.
  static constexpr bool kOwnP = D == 64;            // P beside S, not over it
  static constexpr int kTile = kOwnP ? kBN + kBN / 2 : kBN;  // S (and P) of a tile
  static constexpr int kPCol = kOwnP ? kBN : 0;     // P from S
  static constexpr int kOCol = 2 * kTile;           // then O of both tiles
  static_assert(kOCol + 2 * D <= 512, "tensor memory");
  static constexpr int kOffKv = 2 * kBytes;
  static constexpr int kOffCodes = kOffKv + kSlots * kBytes;
  static constexpr int kOffScale = kOffCodes + kStages * kCodes;    // [kScaleRing][12] of K
  static constexpr int kOffVScale = kOffScale + kScaleRing * 12 * 4;  // [kDualStages][8]
  static constexpr int kOffBar = kOffVScale + kDualStages * 8 * 4;
  static constexpr int kBars = 2 * kSlots + 2 * kDualStages + 2 + 2 + 2 + 4 + 2 + 2 + 2;
  static constexpr int kOffMisc = kOffBar + 8 * kBars;
  static constexpr int kSmem = kOffMisc + 32 + 1024;                // + alignment
  static_assert(kSmem <= 232448, "shared memory");
  static_assert(kStages == kDualStages || 2 * kCodes == kBytes, "two more in a Q tile's place");
  // Where stage s lies.
  static __device__ __forceinline__ uint32_t codes_at(int s) {
    return s < kStages ? kOffCodes + s * kCodes : kBytes + (s - kStages) * kCodes;
  }
};

// Barriers.
template <int D>
struct Bar {
  static constexpr int kFull = 0;
  static constexpr int kEmpty = Tile<D>::kSlots;
  static constexpr int kCodesFull = 2 * Tile<D>::kSlots;
  static constexpr int kCodesEmpty = kCodesFull + Tile<D>::kDualStages;
  static constexpr int kQ = kCodesEmpty + Tile<D>::kDualStages;
  static constexpr int kS = kQ + 2;
  static constexpr int kSRead = kS + 2;   // S is in registers (kOwnP)
  static constexpr int kP = kSRead + 2;   // [tile][part]
  static constexpr int kPV = kP + 4;      // a step's P V has ended (kOwnP)
  static constexpr int kO = kPV + 2;
  static constexpr int kDrain = kO + 2;   // [issuer]
};

// 256 rows of one request and kv head, over steps [step0, step0 + steps) of
// kBN keys: all that they see, or one of `parts` ranges of it.
struct Unit {
  Request rq;
  int request, kvh, row0, rows_in, step0, steps, kv_end;  // kv_end: of this range
  int index;                                              // among all units
  // At most 128 rows: both tiles are these rows, tile i over steps i, i + 2, ...
  bool dual;
};

struct TiledParams : CachedParams {
  int* status;
  unsigned long long timeout_ns;
  int fault_mode;  // 1: nothing is fetched (test of the bounded waits)
  int parts;  // CTAs of a unit; above 1 they leave (max, sum, O) in the workspace
};

// Part `part` of a unit in the workspace, `slots` of them in all: [256][D] f32
// of O, then (max, sum) per row.
template <int D>
struct TilePart {
  static __device__ __forceinline__ float* o(float* ws, long long slot, int row) {
    return ws + (slot * kUnit + row) * D;
  }
  static __device__ __forceinline__ float2* ml(float* ws, long long slots, long long slot, int row) {
    return reinterpret_cast<float2*>(ws + slots * kUnit * D) + slot * kUnit + row;
  }
};

__device__ __forceinline__ long long units_of(const CachedParams& p, const Request& r) {
  const long long rows = static_cast<long long>(r.n) * p.group;
  return rows > p.rows_most ? p.kv_heads * ((rows + kUnit - 1) / kUnit) : 0;
}

// Tokens that a row sees.
__device__ __forceinline__ int row_limit(const CachedParams& p, const Request& rq, int row) {
  const int last = p.causal ? rq.before + row / p.group + 1 : rq.kv;
  return min(max(last, 0), rq.kv);
}

// Unit number `at`.  The requests with most keys come first and, in each,
// the last rows (causal: those that see most), so that the last CTAs to start
// are short; the heads of a row tile follow each other, so that neighbours share
// keys in L2.  (More requests than threads, each with a long prompt: in their
// own order.)  Up to 32 requests: every warp for itself, a lane a request (without
// barriers: 68.4 us on one prompt of 4096, 69.5 with them).
template <bool FROM_L2>
__device__ __forceinline__ bool find_request_few(const CachedParams& p, long long at, Unit& u,
                                                 int& in_request) {
  const int lane = threadIdx.x & 31;
  Request rq{0, 0, 0, 0};
  if (lane < p.batch) rq = request_at<FROM_L2>(p, lane);
  const long long mine = lane < p.batch ? units_of(p, rq) : 0;
  long long before = 0;
  for (int i = 0; i < p.batch; ++i) {
    const int kv = __shfl_sync(~0u, rq.kv, i);
    const long long n = __shfl_sync(~0u, mine, i);
    if (kv > rq.kv || (kv == rq.kv && i < lane)) before += n;
  }
  const unsigned there = __ballot_sync(~0u, at >= before && at < before + mine);
  if (there == 0) return false;
  u.request = __ffs(there) - 1;
  u.rq = Request{__shfl_sync(~0u, rq.start, u.request), __shfl_sync(~0u, rq.n, u.request),
                 __shfl_sync(~0u, rq.kv, u.request), __shfl_sync(~0u, rq.before, u.request)};
  in_request = __shfl_sync(~0u, static_cast<int>(mine - 1 - (at - before)), u.request);
  return true;
}

// The same for any number, by the whole CTA.  `scratch`: 12 bytes a thread.
template <bool FROM_L2>
__device__ __forceinline__ bool find_request(const CachedParams& p, long long at, Unit& u,
                                             int& in_request, uint8_t* scratch) {
  long long* units = reinterpret_cast<long long*>(scratch);
  int* keys = reinterpret_cast<int*>(units + kThreads);
  __shared__ long long where[2];
  const int each = (p.batch + kThreads - 1) / kThreads;
  const int me = static_cast<int>(threadIdx.x);  // of at least kThreads threads
  const int first = me * each, last = min(first + each, p.batch);
  long long mine = 0;
  int kv = 0;
  for (int r = first; r < last; ++r) {
    const Request rq = request_at<FROM_L2>(p, r);
    mine += units_of(p, rq);
    kv = rq.kv;
  }
  units[me] = mine;
  keys[me] = kv;
  if (me == 0) where[0] = -1;
  __syncthreads();
  if (mine > 0) {
    long long before = 0;
    const int threads = min(kThreads, p.batch);
    for (int i = 0; i < threads; ++i) {
      const bool earlier = each == 1 ? keys[i] > kv || (keys[i] == kv && i < me) : i < me;
      if (earlier) before += units[i];
    }
    if (at >= before && at < before + mine) {
      int r = first;
      for (; r + 1 < last; ++r) {
        const long long n = units_of(p, request_at<FROM_L2>(p, r));
        if (at < before + n) break;
        before += n;
      }
      where[0] = r;
      where[1] = units_of(p, request_at<FROM_L2>(p, r)) - 1 - (at - before);
    }
  }
  __syncthreads();
  if (where[0] < 0) return false;
  u.request = static_cast<int>(where[0]);
  u.rq = request_at<FROM_L2>(p, u.request);
  in_request = static_cast<int>(where[1]);
  return true;
}

template <bool FROM_L2 = false>
__device__ bool find_unit(const CachedParams& p, long long at, Unit& u, uint8_t* scratch) {
  int in_request;
  if (!(p.batch <= 32 ? find_request_few<FROM_L2>(p, at, u, in_request)
                      : find_request<FROM_L2>(p, at, u, in_request, scratch)))
    return false;
  u.kvh = in_request % p.kv_heads;
  u.row0 = in_request / p.kv_heads * kUnit;
  u.rows_in = u.rq.n * p.group;
  u.kv_end = row_limit(p, u.rq, min(u.row0 + kUnit, u.rows_in) - 1);
  u.step0 = 0;
  u.steps = (u.kv_end + kBN - 1) / kBN;
  u.index = static_cast<int>(at);
  u.dual = u.rows_in - u.row0 <= kBM && u.steps > 1;
  return true;
}

// Range `part` of `parts` of it.
__device__ __forceinline__ void take_part(Unit& u, int part, int parts) {
  const int each = (u.steps + parts - 1) / parts;
  u.step0 = min(part * each, u.steps);
  u.steps = min(each, u.steps - u.step0);
  u.kv_end = min(u.kv_end, (u.step0 + u.steps) * kBN);
  u.dual = u.dual && u.steps > 1;
}

__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z,
                                             uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}

__device__ __forceinline__ uint32_t mul_half2(uint32_t a, __half2 b) {
  const __half2 h = __hmul2(*reinterpret_cast<__half2*>(&a), b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ---------------------------------------------------------------------------
// Fetching warp: items K_0, V_0, K_1, V_1, ... in 8 bits.  Lane g < 8 fetches
// keys 16 g .. 16 g + 15 of each.  Its K scales go straight to the softmax: the
// place of step j is written again for step j + 8, which waits (through both
// rings, 10 items at most) until S of step j + 3 has ended, and that was issued
// after the softmax had read S, and then the scales, of step j + 1 at least.
// ---------------------------------------------------------------------------
template <int D>
__device__ void fetch_role(const CUtensorMap* map_k, const CUtensorMap* map_v,
                           const TiledParams& p, const Unit& u, uint32_t sbase,
                           const WaitCtx& w) {
  using T = Tile<D>;
  auto bar = [&](int i) { return sbase + T::kOffBar + 8u * i; };
  const int lane = threadIdx.x & 31;
  const int* table = p.tables + u.request * p.table_stride;
  auto id_of = [&](int j) {
    const int key = (u.step0 + j) * kBN + 16 * lane;
    if (lane < 8 && key < u.kv_end) {
      const int id = table[key >> p.shift];
      if (id >= 0 && id < p.num_blocks) return id;
    }
    return -1;
  };
  const int stages = u.dual ? T::kDualStages : T::kStages, shift = stages == 4 ? 2 : 1;
  int sent = 0;
  auto fetch = [&](bool is_v, int j, int id) {
    const int stage = sent & (stages - 1);
    if (!__all_sync(~0u, wait_bar(bar(Bar<D>::kCodesEmpty + stage), ((sent >> shift) & 1) ^ 1, w,
                                  kSiteKvEmpty)))
      return false;
    const uint32_t full = bar(Bar<D>::kCodesFull + stage);
    const int n = __popc(__ballot_sync(~0u, id >= 0));
    // Where the group's scale goes: K's to the softmax, V's to the conversion.
    const uint32_t scale_at =
        sbase + (is_v ? T::kOffVScale + 4 * (8 * stage + lane)
                      : T::kOffScale + 4 * (12 * (j % kScaleRing) + lane));
    if (!is_v) {  // groups whose block is none, bit by bit
      const unsigned holes =
          __ballot_sync(~0u, lane < 8 && id < 0 && (u.step0 + j) * kBN + 16 * lane < u.kv_end);
      if (lane == 0)
        ptx::st_shared_f32(sbase + T::kOffScale + 4 * (12 * (j % kScaleRing) + 8),
                           __uint_as_float(holes));
    }
    if (lane == 0) ptx::mbar_arrive_expect_tx(full, n * T::kGroup);
    __syncwarp();
    if (id >= 0) {
      const int off = ((u.step0 + j) * kBN + 16 * lane) & ((1 << p.shift) - 1);
      const int piece = id * p.kv_heads + u.kvh;
      ptx::tma_load_3d(sbase + T::codes_at(stage) + lane * T::kGroup,
                       is_v ? map_v : map_k, full, 0, D == 128 ? off : off / 2, piece);
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(scale_at),
                   "l"((is_v ? p.vs : p.ks) + piece)
                   : "memory");
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full) : "memory");
    } else if (lane < 8) {
      ptx::st_shared_f32(scale_at, 0.f);
      ptx::mbar_arrive(full);
    }
    ++sent;
    return true;
  };
  int id = id_of(0), next = id_of(1);
  for (int j = 0; j < u.steps; ++j) {
    const int after = id_of(j + 2);
    if (!fetch(false, j, id) || !fetch(true, j, id)) break;
    id = next;
    next = after;
  }
  // After a wait that ran out: copies on their way end before the shared
  // memory that they go to does.
  if (*w.abort) {
    for (int i = max(0, sent - stages); i < sent; ++i) {
      const unsigned long long t0 = ptx::globaltimer_ns();
      while (!ptx::mbar_try_wait(bar(Bar<D>::kCodesFull + (i & (stages - 1))), (i >> shift) & 1) &&
             ptx::globaltimer_ns() - t0 < p.timeout_ns) {
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Converting warpgroup: 8 bits to 16, item by item.
// ---------------------------------------------------------------------------
template <int CODE, int D>
__device__ void convert_role(const TiledParams& p, const Unit& u, uint32_t sbase, uint8_t* sgen,
                             const WaitCtx& w) {
  using T = Tile<D>;
  constexpr int kIters = D / 16;          // 16-byte pieces of codes a thread has of a tile
  constexpr float kVLift = CODE == ATTN_CODE_E4M3 ? 128.f : 256.f;
  auto bar = [&](int i) { return sbase + T::kOffBar + 8u * i; };
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 3;
  float* misc = reinterpret_cast<float*>(sgen + T::kOffMisc);

  // The largest V scale in sight.
  float ref = 0.f;
  const int* table = p.tables + u.request * p.table_stride;
  const int blocks = (u.kv_end + (1 << p.shift) - 1) >> p.shift;
  for (int b = ((u.step0 * kBN) >> p.shift) + 32 * warp + lane; b < blocks; b += 128) {
    const int id = table[b];
    if (id >= 0 && id < p.num_blocks)
      ref = fmaxf(ref, p.vs[static_cast<long long>(id) * p.kv_heads + u.kvh]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) ref = fmaxf(ref, __shfl_xor_sync(~0u, ref, d));
  if (lane == 0) misc[4 + warp] = ref;
  ptx::named_bar_sync(1, 128);
  ref = fmaxf(fmaxf(misc[4], misc[5]), fmaxf(misc[6], misc[7]));
  if (!(ref > 0.f)) ref = 1.f;
  // Scales so small that kVLift / ref would be above the largest f32 (ref below
  // 2^-120) or ref / kVLift below the least normal one: 2^64 times all of them.
  const float up = ref < 0x1p-60f ? 0x1p64f : 1.f;
  ref *= up;
  if (warp == 0 && lane == 0) {
    misc[2] = ref / kVLift;  // what O is multiplied by, and then by this:
    misc[3] = 1.f / up;
  }
  const float to_v = kVLift / ref;

  // A thread's piece `it` of a tile: a row and 16 codes of it, so that the 8
  // lanes of one pass through shared memory meet 8 different 16-byte banks both
  // in the 8-bit tile (16 keys after 16 keys, 128-byte rows) and in the 16-bit
  // one (64-column blocks of 128-byte rows).
  const int row0 = D == 128 ? 4 * warp + 2 * (lane >> 4) + ((lane >> 2) & 1) : 8 * warp + (lane >> 2);
  const int piece = D == 128 ? (lane & 3) + 4 * (((lane >> 2) ^ (lane >> 3)) & 1) : lane & 3;
  constexpr int kRowStep = D == 128 ? 16 : 32;   // rows from one piece to the next
  const int line = D == 128 ? row0 : row0 >> 1;  // 128-byte line of codes
  const int at8 = D == 128 ? piece : (row0 & 1) * 4 + piece;
  const uint32_t codes_at = sbase + line * 128 + ((at8 ^ (line & 7)) << 4);
  const int k16 = (2 * piece) & 7;
  const uint32_t tile_at = sbase + T::kOffKv + (piece >> 2) * T::kBlock + row0 * 128;
  const uint32_t at_lo = (k16 ^ (row0 & 7)) << 4, at_hi = ((k16 + 1) ^ (row0 & 7)) << 4;
  auto group_of = [&](int it) { return D == 128 ? it : 2 * it + (warp >> 1); };

  const int stages = u.dual ? T::kDualStages : T::kStages, shift = stages == 4 ? 2 : 1;
  for (int t = 0; t < 2 * u.steps; ++t) {
    const bool is_v = (t & 1) != 0;
    const int j = t >> 1;
    const int stage = t & (stages - 1), slot = t % T::kSlots;
    bool ok = wait_bar(bar(Bar<D>::kCodesFull + stage), (t >> shift) & 1, w, kSiteKvFull);
    if (!__all_sync(~0u, ok)) return;
    uint32_t c[kIters][4];
#pragma unroll
    for (int it = 0; it < kIters; ++it)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(c[it][0]), "=r"(c[it][1]), "=r"(c[it][2]), "=r"(c[it][3])
                   : "r"(codes_at + T::codes_at(stage) + it * kRowStep * D)
                   : "memory");
    float vs[kIters];
    bool pow2 = true;  // all factors are powers of two that f16 holds, or 0
    if (is_v) {
      const float* scale = reinterpret_cast<const float*>(sgen + T::kOffVScale) + 8 * stage;
#pragma unroll
      for (int it = 0; it < kIters; ++it) {
        vs[it] = scale[group_of(it)] * up * to_v;
        pow2 &= (__float_as_int(vs[it]) & 0x7fffff) == 0 && !(vs[it] > 0.f && vs[it] < 0x1p-24f);
      }
      // What lies behind the last token, or where nothing was fetched, may be
      // any bits: 0 * NaN would reach a sum.  (Among the keys it is masked.)
      const int key0 = (u.step0 + j) * kBN;
      if (key0 + kBN > u.rq.kv) {
#pragma unroll
        for (int it = 0; it < kIters; ++it)
          if (key0 + row0 + it * kRowStep >= u.rq.kv) c[it][0] = c[it][1] = c[it][2] = c[it][3] = 0u;
      }
#pragma unroll
      for (int it = 0; it < kIters; ++it)
        if (vs[it] == 0.f) c[it][0] = c[it][1] = c[it][2] = c[it][3] = 0u;
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(Bar<D>::kCodesEmpty + stage));
    ok = wait_bar(bar(Bar<D>::kEmpty + slot), ((t / T::kSlots) & 1) ^ 1, w, kSiteKvEmpty);
    if (!__all_sync(~0u, ok)) return;
    const uint32_t tile = tile_at + slot * T::kBytes;
    auto store = [&](int it, const uint32_t (&h)[8]) {
      const uint32_t base = tile + it * kRowStep * 128;
      st_shared_v4(base + at_lo, h[0], h[1], h[2], h[3]);
      st_shared_v4(base + at_hi, h[4], h[5], h[6], h[7]);
    };
    auto convert = [&](int it, uint32_t (&h)[8]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[2 * i] = Code<CODE>::half2_lo(c[it][i]);
        h[2 * i + 1] = Code<CODE>::half2_hi(c[it][i]);
      }
    };
    // One branch a tile (asked at each of its 8 pieces: 900 us where this takes 792).
    if (!is_v) {
#pragma unroll
      for (int it = 0; it < kIters; ++it) {
        uint32_t h[8];
        convert(it, h);
        store(it, h);
      }
    } else if (__builtin_expect(pow2, 1)) {
#pragma unroll
      for (int it = 0; it < kIters; ++it) {
        uint32_t h[8];
        convert(it, h);
        const __half2 f2 = __float2half2_rn(vs[it]);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = mul_half2(h[i], f2);
        store(it, h);
      }
    } else {  // scales that the caller brought, or very small ones: one rounding to f16
#pragma unroll
      for (int it = 0; it < kIters; ++it) {
        uint32_t h[8];
        convert(it, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 x = half2_to_float2(h[i]);
          h[i] = half2_of(x.x * vs[it], x.y * vs[it]);
        }
        store(it, h);
      }
    }
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(Bar<D>::kFull + slot));
  }
}

__device__ __forceinline__ uint64_t descriptor(uint32_t lo) {
  constexpr uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "n"(hi));
  return d;
}

// ---------------------------------------------------------------------------
// Issuers.  kOwnP: one thread a tile (`me` = 0, 1), else one for both.
// ---------------------------------------------------------------------------
template <int D>
__device__ void mma_role(const Unit& u, int me, uint32_t tmem, uint32_t sbase, const WaitCtx& w) {
  using T = Tile<D>;
  auto bar = [&](int i) { return sbase + T::kOffBar + 8u * i; };
  constexpr uint32_t kIdescS = ptx::idesc_f16(kBM, kBN, false, false);
  constexpr uint32_t kIdescPV = ptx::idesc_f16(kBM, D, false, true);
  const int tiles = u.rows_in - u.row0 > kBM ? 2 : 1;
  const int n = u.steps;
  auto ring_wait = [&](int t) {
    const bool ok = wait_bar(bar(Bar<D>::kFull + t % T::kSlots), (t / T::kSlots) & 1, w, kSiteKvFull);
    if (ok) ptx::tc_fence_after();
    return ok;
  };
  // Shared memory descriptors: their upper word is the same for all operands
  // (SBO 1024, version 1, 128-byte swizzle), the lower one has the address >> 4
  // and, from bit 16, LBO >> 4 (64-column blocks of V).  Only lower words are
  // kept: with 64-bit ones this thread's registers overflowed into local memory.
  const uint32_t q_lo = (sbase >> 4) | (1u << 16);
  const uint32_t kv_lo = (sbase + T::kOffKv) >> 4;
  auto issue_s = [&](int i, int t) {
    const uint32_t q = q_lo + (u.dual ? 0 : i) * (T::kBytes >> 4);
    const uint32_t k = kv_lo + (t % T::kSlots) * (T::kBytes >> 4) + (1u << 16);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint32_t off = static_cast<uint32_t>((kk >> 2) * T::kBlock + (kk & 3) * 32) >> 4;
      ptx::mma_ss(tmem + i * T::kTile, descriptor(q + off), descriptor(k + off), kIdescS,
                  kk > 0 ? 1u : 0u);
    }
    ptx::mma_commit(bar(Bar<D>::kS + i));
  };
  auto issue_pv = [&](int i, int j, int t, int k0, int k1) {
    const uint32_t v =
        kv_lo + (t % T::kSlots) * (T::kBytes >> 4) + (static_cast<uint32_t>(T::kBlock >> 4) << 16);
#pragma unroll
    for (int kk = k0; kk < k1; ++kk)
      ptx::mma_ts(tmem + T::kOCol + i * D, tmem + i * T::kTile + T::kPCol + kk * 8,
                  descriptor(v + (static_cast<uint32_t>(kk * 2048) >> 4)), kIdescPV,
                  (j > 0 || kk > 0) ? 1u : 0u);
  };
  auto p_wait = [&](int i, int part, int j) {
    const bool ok = wait_bar(bar(Bar<D>::kP + 2 * i + part), j & 1, w, kSitePReady);
    if (ok) ptx::tc_fence_after();
    return ok;
  };

  const int i0 = T::kOwnP ? me : 0, i1 = T::kOwnP ? min(me + 1, tiles) : tiles;
  bool ok = true;
  auto first_s = [&](int i, int t) {
    ok = ring_wait(t) && wait_bar(bar(Bar<D>::kQ + (u.dual ? 0 : i)), 0, w, kSiteQ);
    if (!ok) return;
    ptx::tc_fence_after();
    issue_s(i, t);
  };
  if (u.dual) {
    // Both tiles' steps in turn (kOwnP: one tile's); S of a tile's next step
    // goes behind P V of the present one, or as soon as S has been read.
    const int by = T::kOwnP ? 2 : 1, from = T::kOwnP ? me : 0;
    for (int j = from; j < 2 && ok; j += by) {
      first_s(j, 2 * j);
      if (ok) ptx::mma_commit(bar(Bar<D>::kEmpty + (2 * j) % T::kSlots));
    }
    for (int j = from; j < n && ok; j += by) {
      const int i = j & 1, c = j >> 1, tv = 2 * j + 1, tk = 2 * j + 4;
      const bool more = j + 2 < n;
      if (T::kOwnP && more) {
        if (!(ok = wait_bar(bar(Bar<D>::kSRead + i), c & 1, w, kSiteSFull))) break;
        if (!(ok = ring_wait(tk))) break;
        ptx::tc_fence_after();
        issue_s(i, tk);
        ptx::mma_commit(bar(Bar<D>::kEmpty + tk % T::kSlots));
      }
      if (!(ok = ring_wait(tv))) break;
      if (!(ok = p_wait(i, 0, c))) break;
      issue_pv(i, c, tv, 0, 4);
      if (!T::kOwnP && more && !(ok = ring_wait(tk))) break;
      if (!(ok = p_wait(i, 1, c))) break;
      issue_pv(i, c, tv, 4, 8);
      if (T::kOwnP) {
        ptx::mma_commit(bar(Bar<D>::kPV + i));
      } else if (more) {
        issue_s(i, tk);
        ptx::mma_commit(bar(Bar<D>::kEmpty + tk % T::kSlots));
      } else {
        ptx::mma_commit(bar(Bar<D>::kO + i));
      }
      ptx::mma_commit(bar(Bar<D>::kEmpty + tv % T::kSlots));
    }
  } else if (n > 0 && i0 < i1) {
    for (int i = i0; i < i1 && ok; ++i) first_s(i, 0);
    if (ok) ptx::mma_commit(bar(Bar<D>::kEmpty));
    for (int j = 0; j < n && ok; ++j) {
      const int tv = 2 * j + 1, tk = 2 * j + 2;
      if constexpr (T::kOwnP) {
        const int i = i0;
        if (j + 1 < n) {
          if (!(ok = wait_bar(bar(Bar<D>::kSRead + i), j & 1, w, kSiteSFull))) break;
          if (!(ok = ring_wait(tk))) break;
          ptx::tc_fence_after();
          issue_s(i, tk);
          ptx::mma_commit(bar(Bar<D>::kEmpty + tk % T::kSlots));
        }
        if (!(ok = ring_wait(tv))) break;
        if (!(ok = p_wait(i, 0, j))) break;
        issue_pv(i, j, tv, 0, 4);
        if (!(ok = p_wait(i, 1, j))) break;
        issue_pv(i, j, tv, 4, 8);
        ptx::mma_commit(bar(Bar<D>::kPV + i));
        ptx::mma_commit(bar(Bar<D>::kEmpty + tv % T::kSlots));
      } else {
        if (!(ok = ring_wait(tv))) break;
        for (int i = 0; i < tiles && ok; ++i) {
          if (!(ok = p_wait(i, 0, j))) break;
          issue_pv(i, j, tv, 0, 4);
          if (i == 0 && j + 1 < n && !(ok = ring_wait(tk))) break;
          if (!(ok = p_wait(i, 1, j))) break;
          issue_pv(i, j, tv, 4, 8);
          if (j + 1 < n)
            issue_s(i, tk);  // its commit covers this step's P V too
          else
            ptx::mma_commit(bar(Bar<D>::kO + i));
        }
        if (!ok) break;
        ptx::mma_commit(bar(Bar<D>::kEmpty + tv % T::kSlots));
        if (j + 1 < n) ptx::mma_commit(bar(Bar<D>::kEmpty + tk % T::kSlots));
      }
    }
  }
  // Every MMA issued here has ended before tensor memory is freed.
  ptx::mma_commit(bar(Bar<D>::kDrain + me));
  const unsigned long long t0 = ptx::globaltimer_ns();
  while (!ptx::mbar_try_wait(bar(Bar<D>::kDrain + me), 0)) {
    if (ptx::globaltimer_ns() - t0 > w.timeout_ns) {
      if (w.status) atomicCAS(w.status, 0, kDeviceTimeoutBase + kSiteDrain);
      break;
    }
  }
}

// ---------------------------------------------------------------------------
// Softmax warpgroup of tile i: a thread a row.
// ---------------------------------------------------------------------------
struct Row {
  int r, lane, warp;  // row of the tile (lane of tensor memory), in its warp
  int row, tok, head; // of the request's rows of this kv head; token and query head
  bool live;
};
// A thread's row.  The thread's number is read anew each time, so that what
// only the beginning and the end need takes no registers in the steps between
// (788 -> 784 us on the chunks named above).
__device__ __forceinline__ Row row_of(const CachedParams& p, const Unit& u, int i) {
  int tid;
  asm volatile("mov.u32 %0, %%tid.x;" : "=r"(tid));
  Row x;
  x.lane = tid & 31;
  x.warp = (tid >> 5) & 3;
  x.r = tid & (kBM - 1);
  x.row = u.row0 + (u.dual ? 0 : i * kBM) + x.r;
  x.live = x.row < u.rows_in;
  x.tok = x.live ? x.row / p.group : 0;
  x.head = u.kvh * p.group + (x.live ? x.row - x.tok * p.group : 0);
  return x;
}

template <typename TQ, int D>
__device__ __forceinline__ float load_q(const TiledParams& p, const Unit& u, int i, uint32_t sbase) {
  using T = Tile<D>;
  auto bar = [&](int b) { return sbase + T::kOffBar + 8u * b; };
  const Row x_of = row_of(p, u, i);
  const int lane = x_of.lane, wi = x_of.warp;
  const bool live = x_of.live;
  // Q to shared memory, in f16 (two tiles of the same rows share it).  A warp
  // takes its 32 rows kAtOnce at a time, 16 bytes a lane: rows of a head lie far
  // apart, and threads that read their own rows took up to 15,000 cycles.
  constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kRounds = 32 / kAtOnce;
  const int sub = lane / kLanes, piece = lane % kLanes;
  const uint32_t tile = sbase + i * T::kBytes;
  const uint32_t row_at = tile + (piece >> 3) * T::kBlock + (32 * wi + sub) * 128;
  const TQ* q = static_cast<const TQ*>(p.q) + (u.rq.start + x_of.tok) * p.q_token +
                x_of.head * p.q_head;
  if (!u.dual || i == 0) {
#pragma unroll 1
    for (int it0 = 0; it0 < kRounds; it0 += 8) {
      uint4 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int from = kAtOnce * (it0 + k) + sub;
        const auto at = __shfl_sync(~0u, reinterpret_cast<unsigned long long>(q), from);
        x[k] = __shfl_sync(~0u, live, from) ? __ldg(reinterpret_cast<const uint4*>(at) + piece)
                                            : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at = kAtOnce * (it0 + k) + sub;  // row of the warp's 32
        st_shared_v4(row_at + (it0 + k) * kAtOnce * 128 + (((piece & 7) ^ (at & 7)) << 4), x[k].x,
                     x[k].y, x[k].z, x[k].w);
      }
    }
    __syncwarp();
  }
  float row_f = 1.f;
  if constexpr (std::is_same<TQ, __nv_bfloat16>::value) {
    // bf16: each thread turns its own row, there, into f16 times a power of two.
    const int r = x_of.r;
    auto chunk_at = [&](int c) {
      return tile + (c >> 3) * T::kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    };
    uint32_t y[D / 8][4], top = 0;
    if (!u.dual || i == 0) {
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(y[c][0]), "=r"(y[c][1]), "=r"(y[c][2]), "=r"(y[c][3])
                     : "r"(chunk_at(c))
                     : "memory");
    } else {  // (the other tile has it there; only the power is wanted)
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint4 v = live ? __ldg(reinterpret_cast<const uint4*>(q) + c) : make_uint4(0, 0, 0, 0);
        y[c][0] = v.x;
        y[c][1] = v.y;
        y[c][2] = v.z;
        y[c][3] = v.w;
      }
    }
#pragma unroll
    for (int c = 0; c < D / 8; ++c)
      top = __vmaxu2(top, __vmaxu2(__vmaxu2(y[c][0] & 0x7fff7fffu, y[c][1] & 0x7fff7fffu),
                                   __vmaxu2(y[c][2] & 0x7fff7fffu, y[c][3] & 0x7fff7fffu)));
    top = max(top & 0xffffu, top >> 16);
    const int e = static_cast<int>(top >> 7) - 127;
    const int shift = top > 0 && e < 128 ? max(e - 14, -112) : 0;
    row_f = power_of_two(shift);
    const float inv = power_of_two(-shift);
    if (!u.dual || i == 0) {
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          h[k] = half2_of(__uint_as_float(y[c][k] << 16) * inv,
                          __uint_as_float(y[c][k] & 0xffff0000u) * inv);
        st_shared_v4(chunk_at(c), h[0], h[1], h[2], h[3]);
      }
    }
  }
  if (!u.dual || i == 0) {
    ptx::fence_proxy_async_smem();
    ptx::mbar_arrive(bar(Bar<D>::kQ + i));
  }
  return row_f;
}

template <typename TQ, int D>
__device__ void softmax_role(const TiledParams& p, const Unit& u, int i, uint32_t tmem,
                             uint32_t sbase, const uint8_t* sgen, const WaitCtx& w) {
  using T = Tile<D>;
  auto bar = [&](int b) { return sbase + T::kOffBar + 8u * b; };
  const int lane = threadIdx.x & 31, wi = (threadIdx.x >> 5) & 3;
  const bool tile_there = u.dual || u.row0 + i * kBM < u.rows_in;
  if (!tile_there) return;
  float to_log2 = p.scale_log2;
  if (u.steps > 0) to_log2 *= load_q<TQ, D>(p, u, i, sbase);
  int limit;  // keys of this range that the row sees
  {
    // (rows behind the last one: zeros that see everything, so that they mask nothing)
    const Row x = row_of(p, u, i);
    limit = (x.live ? min(row_limit(p, u.rq, x.row), u.kv_end) : u.kv_end) - u.step0 * kBN;
  }
  const uint32_t lane_base = tmem + (static_cast<uint32_t>(32 * wi) << 16);
  const uint32_t s_col = i * T::kTile, p_col = s_col + T::kPCol, o_col = T::kOCol + i * D;
  float m = -INFINITY, l = 0.f;  // maximum in log2 units, sum of 2^kLift p
  bool ok = true;
  // c counts this tile's steps, j all of them.
  const int by = u.dual ? 2 : 1;
  int c = 0;
  for (int j = u.dual ? i : 0; j < u.steps; j += by, ++c) {
    ok = __all_sync(~0u, wait_bar(bar(Bar<D>::kS + i), c & 1, w, kSiteSFull));
    if (!ok) break;
    ptx::tc_fence_after();
    uint32_t s[kBN];
#pragma unroll
    for (int b = 0; b < kBN / 32; ++b)
      ptx::tmem_ld32(lane_base + s_col + 32 * b, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * b]));
    const int lim = limit - j * kBN;  // columns below it are seen
    // Factors of the groups' scores, and the groups whose block is none.
    float factor[kBN / 16];
    uint32_t holes;
    {
      const uint32_t at = sbase + T::kOffScale + 48 * (j % kScaleRing);
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(factor[0]), "=f"(factor[1]), "=f"(factor[2]), "=f"(factor[3])
                   : "r"(at)
                   : "memory");
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(factor[4]), "=f"(factor[5]), "=f"(factor[6]), "=f"(factor[7])
                   : "r"(at + 16)
                   : "memory");
      holes = __float_as_uint(ptx::ld_shared_f32(at + 32));
    }
#pragma unroll
    for (int g = 0; g < kBN / 16; ++g) factor[g] *= to_log2;
    ptx::tmem_wait_ld();
    ptx::reg_fence(s);
    if constexpr (T::kOwnP) {  // the next S may come
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(Bar<D>::kSRead + i));
    }
    if (__any_sync(~0u, lim < kBN) || holes != 0) {
#pragma unroll
      for (int k = 0; k < kBN; ++k)
        if (k >= lim || ((holes >> (k / 16)) & 1u)) s[k] = __float_as_uint(-INFINITY);
      // The factor of a group which the row does not see may be anything (NaN):
      // 1 keeps -inf there.  The least factor keeps -inf too, where the product
      // above may reach 0 (f16 products are below 2^32, so scores that small
      // are 0 either way); NaN stays.
#pragma unroll
      for (int g = 0; g < kBN / 16; ++g) {
        if (factor[g] < 0x1p-90f) factor[g] = 0x1p-90f;
        if (16 * g >= lim || ((holes >> g) & 1u)) factor[g] = 1.f;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < kBN / 16; ++g) {
      float a[5];
#pragma unroll
      for (int k = 0; k < 5; ++k)
        a[k] = ptx::fmax3(__uint_as_float(s[16 * g + 3 * k]), __uint_as_float(s[16 * g + 3 * k + 1]),
                          __uint_as_float(s[16 * g + 3 * k + 2]));
      const float b = ptx::fmax3(a[0], a[1], a[2]);
      const float d = ptx::fmax3(a[3], a[4], __uint_as_float(s[16 * g + 15]));
      top = fmaxf(top, fmaxf(b, d) * factor[g]);
    }
    float alpha = 1.f;
    bool move = false;
    if (c == 0) {
      m = top;
    } else if (top - m > kMove) {
      alpha = ptx::ex2_approx(m - top);
      m = top;
      move = true;
    }
    // The last step's P V has ended: O has the sum so far, P's columns are free.
    // (P over S: S was issued behind that P V, so its commit said so.)
    bool waited = !T::kOwnP || c == 0;
    auto pv_wait = [&]() {
      if (!waited) {
        ok = __all_sync(~0u, wait_bar(bar(Bar<D>::kPV + i), (c - 1) & 1, w, kSiteODone));
        ptx::tc_fence_after();
        waited = true;
      }
    };
    if (__any_sync(~0u, move)) {
      pv_wait();
#pragma unroll 1
      for (int b = 0; b < D / 32; ++b) {
        uint32_t o[32];
        ptx::tmem_ld32(lane_base + o_col + 32 * b, o);
        ptx::tmem_wait_ld();
        ptx::reg_fence(o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
        ptx::tmem_st32(lane_base + o_col + 32 * b, o);
      }
    }
    const float neg = m == -INFINITY ? 0.f : kLift - m;
    const uint64_t neg2 = ptx::f2_pack(neg, neg);
    uint64_t part[2] = {0ull, 0ull};
    // A batch's exponentials are asked for before the last batch's are used, and
    // where P has columns of its own the first 32 wait in registers for the last
    // step's P V: 70.5 -> 69.4 us on a prompt of 4096, 16 heads of 64 (batches of
    // 2 pairs 70.4, of 16 69.6); at D = 128 no difference.
    constexpr int kBatch = 8;  // pairs
    uint32_t pk[2][16];
    float before[2 * kBatch];
#pragma unroll
    for (int at = 0; at <= kBN / 2; at += kBatch) {
      float x[2 * kBatch];
      if (at < kBN / 2) {
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const int c0 = 2 * (at + e);
          const float f = factor[c0 / 16];
          const uint64_t x2 = ptx::f2_fma(
              ptx::f2_pack(__uint_as_float(s[c0]), __uint_as_float(s[c0 + 1])), ptx::f2_pack(f, f),
              neg2);
          ptx::f2_unpack(x2, x[2 * e], x[2 * e + 1]);
        }
#pragma unroll
        for (int e = 0; e < 2 * kBatch; ++e) x[e] = ptx::ex2_approx(x[e]);
      }
      if (at > 0) {
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const int k = at - kBatch + e;
          part[e & 1] = ptx::f2_add(part[e & 1], ptx::f2_pack(before[2 * e], before[2 * e + 1]));
          pk[(k / 16) & 1][k % 16] = half2_of(before[2 * e], before[2 * e + 1]);
        }
        if (at == 16 && !T::kOwnP) ptx::tmem_st16(lane_base + p_col, pk[0]);
        if (at == 32) {
          if (T::kOwnP) {
            pv_wait();
            ptx::tmem_st16(lane_base + p_col, pk[0]);
          }
          ptx::tmem_st16(lane_base + p_col + 16, pk[1]);
          ptx::tmem_wait_st();  // P V of 64 keys may begin
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(Bar<D>::kP + 2 * i));
        }
        if (at == 48) ptx::tmem_st16(lane_base + p_col + 32, pk[0]);
        if (at == 64) ptx::tmem_st16(lane_base + p_col + 48, pk[1]);
      }
#pragma unroll
      for (int e = 0; e < 2 * kBatch; ++e) before[e] = x[e];
    }
    ptx::tmem_wait_st();
    ptx::tc_fence_before();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(Bar<D>::kP + 2 * i + 1));
    float sa, sb, sc, sd;
    ptx::f2_unpack(part[0], sa, sb);
    ptx::f2_unpack(part[1], sc, sd);
    l = l * alpha + ((sa + sb) + (sc + sd));
  }

  float f = 0.f, down = 1.f;
  if (u.steps > 0) {
    if (ok) {
      const bool done = T::kOwnP ? wait_bar(bar(Bar<D>::kPV + i), (c - 1) & 1, w, kSiteODone)
                                 : wait_bar(bar(Bar<D>::kO + i), 0, w, kSiteODone);
      ok = __all_sync(~0u, done);
      ptx::tc_fence_after();
    }
    f = reinterpret_cast<const float*>(sgen + T::kOffMisc)[2];
    down = reinterpret_cast<const float*>(sgen + T::kOffMisc)[3];
  }
  // Two tiles of the same rows: tile 1 hands its sums over in the rings' place,
  // once both have no MMA left that reads there; tile 0 adds them to its own.
  const Row x_of = row_of(p, u, i);
  const int r = x_of.r;
  const bool live = x_of.live;
  float other = 0.f;
  float4* hand = reinterpret_cast<float4*>(const_cast<uint8_t*>(sgen) + T::kOffKv) + r;
  if (u.dual) {
    float2* hand_ml = reinterpret_cast<float2*>(hand - r + kBM * (D / 4)) + r;
    ptx::named_bar_sync(2, 2 * kBM);
    if (i == 1) {
#pragma unroll 1
      for (int b = 0; b < D / 32; ++b) {
        uint32_t o[32];
        ptx::tmem_ld32(lane_base + o_col + 32 * b, o);
        ptx::tmem_wait_ld();
        ptx::reg_fence(o);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          hand[(8 * b + k) * kBM] =
              make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                          __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
      }
      *hand_ml = make_float2(m, l);
    }
    ptx::named_bar_sync(2, 2 * kBM);
    if (i == 1) return;
    const float2 ml = *hand_ml;
    const float now = fmaxf(m, ml.x), base = now == -INFINITY ? 0.f : now;
    const float mine = ptx::ex2_approx(m - base);
    other = ptx::ex2_approx(ml.x - base) * f;
    f *= mine;
    l = l * mine + ml.y * ptx::ex2_approx(ml.x - base);
    m = now;
  }
  if (!ok) return;
  if (p.parts == 1 && u.steps > 0) {
    const float n = m == -INFINITY && l == l ? 0.f : 1.f / l;
    f *= n;
    other *= n;
  }
  TQ* out = static_cast<TQ*>(p.out) + (u.rq.start + x_of.tok) * p.o_token +
            x_of.head * p.o_head;
  const long long slots = gridDim.x, slot = blockIdx.x;
  float* o_part = TilePart<D>::o(p.ws, slot, i * kBM + r);
  if (p.parts > 1 && live)
    *TilePart<D>::ml(p.ws, slots, slot, i * kBM + r) = make_float2(m, u.steps > 0 ? l : 0.f);
#pragma unroll 1
  for (int b = 0; b < D / 32; ++b) {
    uint32_t o[32];
    if (u.steps > 0) {
      ptx::tmem_ld32(lane_base + o_col + 32 * b, o);
      ptx::tmem_wait_ld();
      ptx::reg_fence(o);
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0u;
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
    if (u.dual) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float4 y = hand[(8 * b + k) * kBM];
        o[4 * k] = __float_as_uint(fmaf(y.x, other, __uint_as_float(o[4 * k])));
        o[4 * k + 1] = __float_as_uint(fmaf(y.y, other, __uint_as_float(o[4 * k + 1])));
        o[4 * k + 2] = __float_as_uint(fmaf(y.z, other, __uint_as_float(o[4 * k + 2])));
        o[4 * k + 3] = __float_as_uint(fmaf(y.w, other, __uint_as_float(o[4 * k + 3])));
      }
    }
    if (down != 1.f) {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * down);
    }
    if (p.parts > 1) {
      if (!live) continue;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        *reinterpret_cast<float4*>(o_part + 32 * b + 4 * k) = make_float4(
            __uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
            __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
      continue;
    }
    // Through the place of this tile's Q, which no MMA reads any more.
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = pack2<TQ>(__uint_as_float(o[8 * k + 2 * e]), __uint_as_float(o[8 * k + 2 * e + 1]));
      const int chunk = 4 * b + k;
      st_shared_v4(sbase + i * T::kBytes + (chunk >> 3) * T::kBlock + r * 128 +
                       (((chunk & 7) ^ (r & 7)) << 4),
                   y[0], y[1], y[2], y[3]);
    }
  }
  if (p.parts > 1) return;
  constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kRounds = 32 / kAtOnce;
  const int sub = x_of.lane / kLanes, piece = x_of.lane % kLanes;
  const uint32_t row_at =
      sbase + i * T::kBytes + (piece >> 3) * T::kBlock + (32 * x_of.warp + sub) * 128;
  __syncwarp();
#pragma unroll 4
  for (int it = 0; it < kRounds; ++it) {
    const int at = kAtOnce * it + sub;
    const auto dst = __shfl_sync(~0u, reinterpret_cast<unsigned long long>(out), at);
    uint4 y;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                 : "r"(row_at + it * kAtOnce * 128 + (((piece & 7) ^ (at & 7)) << 4))
                 : "memory");
    if (__shfl_sync(~0u, live, at)) reinterpret_cast<uint4*>(dst)[piece] = y;
  }
}

// Joins the parts of unit blockIdx.x, rows 16 blockIdx.y .. + 15: a warp a row.
template <typename TQ, int D>
__global__ void __launch_bounds__(kThreads) join_kernel(const TiledParams p) {
  __shared__ __align__(16) uint8_t scratch[12 * kThreads];
  Unit u;
  const bool there = find_unit<true>(p, blockIdx.x, u, scratch);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!there) return;
  const int lane = threadIdx.x & 31, r = 16 * blockIdx.y + (threadIdx.x >> 5);
  const int row = u.row0 + r;
  if (row >= u.rows_in) return;
  const long long slots = static_cast<long long>(gridDim.x) * p.parts;
  constexpr int kPer = D / 32;
  float top = -INFINITY, sum = 0.f, x[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) x[e] = 0.f;
#pragma unroll 4
  for (int part = 0; part < p.parts; ++part) {
    const long long slot = static_cast<long long>(u.index) * p.parts + part;
    const float2 ml = *TilePart<D>::ml(p.ws, slots, slot, r);
    const float* o = TilePart<D>::o(p.ws, slot, r) + lane * kPer;
    float y[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) y[e] = o[e];
    const float now = fmaxf(top, ml.x), base = now == -INFINITY ? 0.f : now;
    const float a = ptx::ex2_approx(top - base), b = ptx::ex2_approx(ml.x - base);
    top = now;
    sum = sum * a + ml.y * b;
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = x[e] * a + y[e] * b;
  }
  const float n = top == -INFINITY && sum == sum ? 0.f : 1.f / sum;
  const int tok = row / p.group;
  TQ* out = static_cast<TQ*>(p.out) + (u.rq.start + tok) * p.o_token +
            (u.kvh * p.group + row - tok * p.group) * p.o_head + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; e += 2)
    *reinterpret_cast<uint32_t*>(out + e) = pack2<TQ>(x[e] * n, x[e + 1] * n);
}

template <typename TQ, int CODE, int D>
__global__ void __launch_bounds__(kThreads, 1)
tiled_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
             const TiledParams p) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL)
  using T = Tile<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Unit u;
  asm volatile("griddepcontrol.launch_dependents;");
  if (!find_unit(p, blockIdx.x / p.parts, u, sgen)) return;
  if (p.parts > 1) take_part(u, blockIdx.x % p.parts, p.parts);

  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sgen + T::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sgen + T::kOffMisc + 4);
  if (threadIdx.x == 0) {
    auto bar = [&](int i) { return sbase + T::kOffBar + 8u * i; };
    for (int s = 0; s < T::kSlots; ++s) {
      ptx::mbar_init(bar(Bar<D>::kFull + s), 4);
      ptx::mbar_init(bar(Bar<D>::kEmpty + s),
                     T::kOwnP && u.rows_in - u.row0 > kBM ? 2 : 1);  // issuers that read it
    }
    for (int s = 0; s < T::kDualStages; ++s) {
      ptx::mbar_init(bar(Bar<D>::kCodesFull + s), 8 + 1);
      ptx::mbar_init(bar(Bar<D>::kCodesEmpty + s), 4);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar(Bar<D>::kQ + i), kBM);
      ptx::mbar_init(bar(Bar<D>::kS + i), 1);
      ptx::mbar_init(bar(Bar<D>::kP + 2 * i), 4);
      ptx::mbar_init(bar(Bar<D>::kP + 2 * i + 1), 4);
      ptx::mbar_init(bar(Bar<D>::kO + i), 1);
      ptx::mbar_init(bar(Bar<D>::kSRead + i), 4);
      ptx::mbar_init(bar(Bar<D>::kPV + i), 1);
      ptx::mbar_init(bar(Bar<D>::kDrain + i), 1);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 12) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const WaitCtx w{abort_flag, p.status, p.timeout_ns};

  // Registers of the four warpgroups: 128 x (2 * 184 + 80 + 64) = 512 * 128.
  if (warp < 8) {
    ptx::setmaxnreg_inc<184>();
    softmax_role<TQ, D>(p, u, warp >> 2, tmem, sbase, sgen, w);
  } else if (warp < 12) {
    ptx::setmaxnreg_dec<80>();
    convert_role<CODE, D>(p, u, sbase, sgen, w);
  } else {
    ptx::setmaxnreg_dec<64>();
    if ((warp == 12 || (T::kOwnP && warp == 14)) && lane == 0)
      mma_role<D>(u, warp == 12 ? 0 : 1, tmem, sbase, w);
    if (warp == 13 && p.fault_mode == 0) fetch_role<D>(&map_k, &map_v, p, u, sbase, w);
    __syncwarp();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
#endif
}

template <typename TQ, int CODE, int D>
int launch(const TiledParams& p, long long units, cudaStream_t st) {
  auto kern = tiled_kernel<TQ, CODE, D>;
  CUtensorMap map_k, map_v;
  if (const int e = codes_map(&map_k, p.kc, p, D)) return e;
  if (const int e = codes_map(&map_v, p.vc, p, D)) return e;
  // Once per device (setting it again does no harm).
  static std::atomic<bool> set_up[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ATTN_ERR_CUDA;
  if (dev >= 64 || !set_up[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Tile<D>::kSmem) != cudaSuccess)
      return ATTN_ERR_RESOURCE;
    if (dev < 64) set_up[dev].store(true, std::memory_order_release);
  }
  kern<<<static_cast<unsigned>(units * p.parts), kThreads, Tile<D>::kSmem, st>>>(map_k, map_v, p);
  if (cudaGetLastError() != cudaSuccess) return ATTN_ERR_CUDA;
  if (p.parts == 1) return ATTN_OK;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(units), kUnit / 16);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<TQ, D>, p) == cudaSuccess ? ATTN_OK : ATTN_ERR_CUDA;
}

template <typename TQ, int CODE>
int launch_d(const TiledParams& p, int D, long long units, cudaStream_t st) {
  return D == 64 ? launch<TQ, CODE, 64>(p, units, st) : launch<TQ, CODE, 128>(p, units, st);
}

template <typename TQ>
int launch_code(const TiledParams& p, int D, int code, long long units, cudaStream_t st) {
  return code == ATTN_CODE_E4M3 ? launch_d<TQ, ATTN_CODE_E4M3>(p, D, units, st)
                                : launch_d<TQ, ATTN_CODE_INT8>(p, D, units, st);
}

// Steps that a range of keys has at least, where the table allows for more.
constexpr int kLeastSteps = 8;

int most_parts(int capacity) {
  const int n = (capacity + kLeastSteps * kBN - 1) / (kLeastSteps * kBN);
  return n > 1 ? n : 1;
}

size_t part_bytes(int D) { return sizeof(float) * kUnit * (D + 2); }

int sm_count(int* sms) {
  static std::atomic<int> known[64];  // per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ATTN_ERR_CUDA;
  int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return ATTN_ERR_CUDA;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  *sms = n;
  return ATTN_OK;
}

}  // namespace

int launch_tiled(const CachedParams& q, int D, int dtype, int code, void* ws,
                 unsigned long long ws_bytes, cudaStream_t st) {
  TiledParams p;
  static_cast<CachedParams&>(p) = q;
  p.status = device_status_ptr();
  if (p.status == nullptr) return ATTN_ERR_CUDA;
  p.timeout_ns = current_timeout_ns();
  p.fault_mode = current_fault_mode();
  // Each request's rows end in at most one unit that is not full.
  const long long rows = static_cast<long long>(p.tokens) * p.group;
  const long long units =
      p.kv_heads * (p.batch == 1 ? (rows + kUnit - 1) / kUnit : rows / kUnit + p.batch);
  if (units > INT_MAX) return ATTN_ERR_INVALID_ARG;
  // Fewer units than SMs: their keys are cut so that every SM has some, but
  // into no more ranges than leave each kLeastSteps steps.
  int sms = 0;
  if (const int e = sm_count(&sms)) return e;
  const int most = most_parts(p.capacity);
  p.parts = static_cast<int>(units > 0 && units < sms ? sms / units : 1);
  if (p.parts > most) p.parts = most;
  if (p.parts > 1 && (ws == nullptr || ws_bytes < part_bytes(D) * units * p.parts))
    return ATTN_ERR_WORKSPACE;
  p.ws = static_cast<float*>(ws);
  return dtype == ATTN_DTYPE_F16 ? launch_code<__half>(p, D, code, units, st)
                                 : launch_code<__nv_bfloat16>(p, D, code, units, st);
}

int tiled_workspace(int D, int capacity, unsigned long long* bytes) {
  *bytes = 0;
  if (most_parts(capacity) == 1) return ATTN_OK;
  int sms = 0;
  if (const int e = sm_count(&sms)) return e;
  *bytes = part_bytes(D) * sms;
  return ATTN_OK;
}

}  // namespace cache
}  // namespace attnprof
