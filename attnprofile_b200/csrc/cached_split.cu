// Attention over the 8-bit cache for few query rows a request (single tokens,
// drafts): every key and value is read once from HBM, so the bytes of the
// codes bound it.
//
// Work.  A unit is 8 NT query rows (token x head of the group) of one request
// and kv head, over chunks of 256 keys; all units' chunks, in order, are cut
// into equal ranges, one a CTA, whatever the requests' lengths.  A range may
// hold parts of two units and any number of whole ones; whole units are
// written at once, parts go to the workspace as (max, sum, O) and a second
// kernel joins them in the order of the keys, so results do not depend on which
// CTA came first.  The ranges are found by every CTA from the lengths alone.
//
// Inside a CTA four warps take 64 keys of a chunk each.  S^T = K Q^T and
// O^T = V^T P^T run on m16n8k16 MMAs with the keys (then the head dimension)
// on the 16 side and 8 query rows on the other, so that the 1 to 8 rows of a
// decode step waste nothing; tcgen05's smallest tile of 64 to 128 rows would be
// almost empty, and its operands would have to go through shared memory in 16
// bits.  Codes go from global memory straight into registers: which key or
// which head dimension a lane holds is free in a contraction as long as both
// operands agree, so lanes take 16 bytes of a row and convert them in place.
// K's scale multiplies the scores in f32; V's scale multiplies each block's
// sum of p v in f32, so no scale is rounded.  P is rounded to f16, by at most
// 2^-11 of itself as an f16 result is (a bf16 result by 2^-8): it is held as
// 2^15 p, in [0, 2^15], so that also weights down to 2^-29 of the largest keep
// all their bits.  Maximum, sum and O are f32.  bf16 queries become f16 times a
// power of two per row, which loses nothing above 2^-38 of the row's largest.
#include <climits>

#include "cached_attn.cuh"
#include "ptx.cuh"

namespace attnprof {
namespace cache {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kChunk = 256;                  // keys
constexpr int kWarpKeys = kChunk / kWarps;   // keys of a chunk that a warp takes
constexpr float kLift = 15.f;                // P is held as 2^kLift p

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

// 16 or 8 bytes of codes (a lane's share of one row).
template <int WORDS>
struct Words {
  uint32_t w[WORDS];
};
template <int WORDS>
__device__ __forceinline__ void load_codes(Words<WORDS>& d, const uint8_t* p) {
  if constexpr (WORDS == 4) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    d.w[0] = v.x; d.w[1] = v.y; d.w[2] = v.z; d.w[3] = v.w;
  } else {
    const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
    d.w[0] = v.x; d.w[1] = v.y;
  }
}

// ---------------------------------------------------------------------------
// The cut of all work into ranges.
// ---------------------------------------------------------------------------
struct Shape {
  int units, chunks;  // of one request: its units, and the chunks of each
};

template <int NT>
__device__ __forceinline__ Shape shape_of(const CachedParams& p, const Request& r) {
  const long long rows = static_cast<long long>(r.n) * p.group;
  if (rows == 0 || rows > p.rows_most) return Shape{0, 1};
  return Shape{p.kv_heads * static_cast<int>((rows + 8 * NT - 1) / (8 * NT)),
               max(1, (r.kv + kChunk - 1) / kChunk)};
}

struct Place {
  int request;
  long long before;  // chunks of all requests in front of it
};

// Sum of all requests' chunks; a place in them is looked up afterwards: each
// thread keeps the sum of its share of the requests.
template <int NT>
__device__ __forceinline__ long long count_chunks(const CachedParams& p, long long* part) {
  const int each = (p.batch + blockDim.x - 1) / blockDim.x;
  const int first = static_cast<int>(threadIdx.x) * each;
  long long sum = 0;
  for (int r = first; r < min(first + each, p.batch); ++r) {
    const Shape s = shape_of<NT>(p, request_at(p, r));
    sum += static_cast<long long>(s.units) * s.chunks;
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

// The request that holds chunk `at` (at < the total); by one thread.
template <int NT>
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
    const Shape s = shape_of<NT>(p, request_at(p, pl.request));
    const long long w = static_cast<long long>(s.units) * s.chunks;
    if (pl.before + w > at || pl.request + 1 >= p.batch) return pl;
    pl.before += w;
    ++pl.request;
  }
}

__device__ __forceinline__ long long chunks_each(long long total) {
  return (total + gridDim.x - 1) / gridDim.x;
}

// Where a part of CTA `cta` lies in the workspace: slot 1 for the part that
// begins its unit, slot 0 for one that begins inside it.  [rows][D] f32 of O
// for all slots, then (max, sum) per row.
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
// One warp's share of a part: the online softmax over its keys.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ uint32_t pack_out(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_out<__half>(float a, float b) { return pack_half2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack_out<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int CODE, int D, int NT>
__global__ void __launch_bounds__(kThreads) split_kernel(const CachedParams p) {
  constexpr int kRows = 8 * NT;
  constexpr int KSTEPS = D / 16;               // MMAs along the head dimension
  constexpr int MT = D / 16;                   // 16-row tiles of O^T
  constexpr int VW = D / 32;                   // words of a V row that a lane holds (D / 8 bytes)
  constexpr int KP = D / 64;                   // 16-byte pieces of a K row that a lane holds
  constexpr bool kQShared = NT >= 4;           // Q operands from shared memory, to save registers
  constexpr int KT = NT >= 4 ? 1 : 2;          // 16-key tiles of one step
  constexpr int kStep = 16 * KT;

  __shared__ long long part_sum[kThreads];
  __shared__ Place place;
  __shared__ float row_m[kWarps][kRows], row_l[kWarps][kRows];
  extern __shared__ float smem[];              // [kWarps][kRows][D + 4] f32, then Q operands
  constexpr int kPitch = D + 4;
  uint2* q_sh = reinterpret_cast<uint2*>(smem + kWarps * kRows * kPitch);

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;

  const long long total = count_chunks<NT>(p, part_sum);
  const long long each = chunks_each(total);
  long long at = each * blockIdx.x;
  const long long stop = min(at + each, total);
  asm volatile("griddepcontrol.launch_dependents;");
  if (at >= stop) return;
  if (threadIdx.x == 0) place = find_place<NT>(p, part_sum, at);
  __syncthreads();
  Place pl = place;

  while (at < stop) {
    const Request rq = request_at(p, pl.request);
    const Shape sh = shape_of<NT>(p, rq);
    const long long work = static_cast<long long>(sh.units) * sh.chunks;
    if (at >= pl.before + work) {
      pl.before += work;
      if (++pl.request >= p.batch) return;
      continue;
    }
    const long long in = at - pl.before;
    const int unit = static_cast<int>(in / sh.chunks);
    const int c0 = static_cast<int>(in - static_cast<long long>(unit) * sh.chunks);
    const int c1 = static_cast<int>(min(static_cast<long long>(sh.chunks), c0 + (stop - at)));
    const int tiles = sh.units / p.kv_heads;
    const int kvh = unit / tiles;
    const int row0 = (unit - kvh * tiles) * kRows;  // of the request's rows of this kv head
    const int rows_in = rq.n * p.group;

    // Q operands: lane (g, t) holds row 8 nt + g, the head dimensions that its
    // K bytes belong to.
    uint32_t qb[kQShared ? 1 : NT][kQShared ? 1 : KSTEPS][2];
    float row_f[NT][2];  // score factor of rows 2t, 2t + 1
    int limit[NT][2];    // keys that they see
    int least = INT_MAX;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + 8 * nt + g;
      const bool live = row < rows_in;
      const int tok = live ? row / p.group : 0;
      const T* qr = static_cast<const T*>(p.q) + (rq.start + tok) * p.q_token +
                    (kvh * p.group + (live ? row - tok * p.group : 0)) * p.q_head;
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
        if (top > 0 && e < 128) f = power_of_two(min(max(e - 14, -112), 112));
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
            b.x = pack_half2(to_float(qr[d]) * inv, to_float(qr[d + 1]) * inv);
            b.y = pack_half2(to_float(qr[d + 2]) * inv, to_float(qr[d + 3]) * inv);
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
        const int r = row0 + 8 * nt + 2 * t + j;
        // (rows behind the last one: zeros that see everything)
        limit[nt][j] = r < rows_in && p.causal ? rq.kv - rq.n + r / p.group + 1 : rq.kv;
        limit[nt][j] = min(limit[nt][j], rq.kv);
        least = min(least, limit[nt][j]);
      }
    }
    least = __reduce_min_sync(~0u, least);
    if constexpr (kQShared) __syncthreads();

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

    // This warp's steps: kWarpKeys / kStep of them in each chunk.
    const int* table = p.tables + pl.request * p.table_stride;
    constexpr int kPerChunk = kWarpKeys / kStep;
    const int steps = (c1 - c0) * kPerChunk;
    auto key_of = [&](int s) {
      return (c0 + s / kPerChunk) * kChunk + warp * kWarpKeys + (s % kPerChunk) * kStep;
    };
    // Block of each 16-key tile of step s (-1: no keys there, or not a block).
    auto blocks_of = [&](int s, int (&id)[KT]) {
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const int key = key_of(s) + 16 * k;
        id[k] = -1;
        if (s < steps && key < rq.kv) {
          const int b = table[key >> p.shift];
          if (b >= 0 && b < p.num_blocks) id[k] = b;
        }
      }
    };
    Words<4> kw[KT][2][KP];   // [tile][row g, row g + 8][piece]
    Words<VW> vw[KT][4];      // [tile][keys 2t, 2t + 1, 2t + 8, 2t + 9]
    float ksc[KT], vsc[KT];
    auto tile_at = [&](int s, int k, int id) {
      const int off = (key_of(s) + 16 * k) & ((1 << p.shift) - 1);
      return ((((static_cast<long long>(id) * p.kv_heads + kvh) << p.shift) + off)) * D;
    };
    // Codes are read also behind the request's last token, within its block;
    // what lies there does not count (masked; V codes are zeroed).
    auto load_k = [&](int s, const int (&id)[KT]) {
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        if (id[k] >= 0) {
          const uint8_t* b = p.kc + tile_at(s, k, id[k]);
          ksc[k] = p.ks[static_cast<long long>(id[k]) * p.kv_heads + kvh];
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int pc = 0; pc < KP; ++pc)
              load_codes(kw[k][r][pc], b + (g + 8 * r) * D + 64 * pc + 16 * t);
        } else {
          ksc[k] = 0.f;
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int pc = 0; pc < KP; ++pc)
#pragma unroll
              for (int i = 0; i < 4; ++i) kw[k][r][pc].w[i] = 0u;
        }
      }
    };
    auto load_v = [&](int s, const int (&id)[KT]) {
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        if (id[k] >= 0) {
          const uint8_t* b = p.vc + tile_at(s, k, id[k]);
          vsc[k] = p.vs[static_cast<long long>(id[k]) * p.kv_heads + kvh];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            load_codes(vw[k][r], b + (2 * t + (r & 1) + 8 * (r >> 1)) * D + 4 * VW * g);
        } else {
          vsc[k] = 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < VW; ++i) vw[k][r].w[i] = 0u;
        }
      }
    };

    int id[KT], id_next[KT];
    blocks_of(0, id);
    load_k(0, id);
    load_v(0, id);
    blocks_of(1, id_next);

    for (int s = 0; s < steps; ++s) {
      const int key0 = key_of(s);
      // S^T = K Q^T
      float sc[NT][KT][4];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][k][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
          const uint32_t w0 = kw[k][0][ks / 4].w[ks % 4], w1 = kw[k][1][ks / 4].w[ks % 4];
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
      float kscale[KT];
      bool held[KT];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        kscale[k] = ksc[k];
        held[k] = id[k] >= 0;
      }
      load_k(s + 1, id_next);

      // Scores in log2 units, masked; the running maximum.
      const bool whole = key0 + kStep <= least;
      bool moved = false;
      float alpha[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = -INFINITY;
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            const float f = kscale[k] * row_f[nt][j];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x = sc[nt][k][2 * h + j] * f;
              if (!held[k] || (!whole && key0 + 16 * k + 8 * h + g >= limit[nt][j])) x = -INFINITY;
              sc[nt][k][2 * h + j] = x;
              top = fmaxf(top, x);
            }
          }
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
          const float now = fmaxf(m[nt][j], top);
          const float base = now == -INFINITY ? 0.f : now - kLift;
          alpha[nt][j] = ptx::ex2_approx(m[nt][j] - kLift - base);
          moved |= now != m[nt][j];
          m[nt][j] = now;
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float e = ptx::ex2_approx(sc[nt][k][2 * h + j] - base);
              sc[nt][k][2 * h + j] = e;
              sum += e;
            }
          l[nt][j] = l[nt][j] * alpha[nt][j] + sum;
        }
      if (__any_sync(~0u, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][mt][i] *= alpha[nt][i & 1];
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
      // Codes behind the last token may be any bits, NaN among them.
      if (key0 + kStep > rq.kv) {
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + 16 * k + 2 * t + (r & 1) + 8 * (r >> 1) >= rq.kv)
#pragma unroll
              for (int i = 0; i < VW; ++i) vw[k][r].w[i] = 0u;
      }
      // O^T += scale (V^T P^T), the scale once a block: tiles of one block add up first.
      // (Their scale is the first one's: the second may have no token.)
      const bool joint = KT == 2 && p.shift > 4;
#pragma unroll
      for (int mp = 0; mp < MT / 2; ++mp) {
        float acc[2][NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[h][nt][i] = 0.f;
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
          if (!joint || k == KT - 1) {
            const float f = joint ? vsc[0] : vsc[k];
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
      load_v(s + 1, id_next);
#pragma unroll
      for (int k = 0; k < KT; ++k) id[k] = id_next[k];
      blocks_of(s + 2, id_next);
    }

    // The four warps' results together.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float s = l[nt][j];
        s += __shfl_xor_sync(~0u, s, 4);
        s += __shfl_xor_sync(~0u, s, 8);
        s += __shfl_xor_sync(~0u, s, 16);
        if (g == 0) {
          row_m[warp][8 * nt + 2 * t + j] = m[nt][j];
          row_l[warp][8 * nt + 2 * t + j] = s;
        }
        float* dst = smem + (warp * kRows + 8 * nt + 2 * t + j) * kPitch + 4 * VW * g;
#pragma unroll
        for (int mt = 0; mt < MT; mt += 2)
          *reinterpret_cast<float4*>(dst + 2 * mt) =
              make_float4(o[nt][mt][j], o[nt][mt][2 + j], o[nt][mt + 1][j], o[nt][mt + 1][2 + j]);
      }
    __syncthreads();
    const bool all_keys = c0 == 0 && c1 == sh.chunks;
    const long long slot = 2ll * blockIdx.x + (c0 == 0 ? 1 : 0);
    for (int i = threadIdx.x; i < kRows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = 4 * (i % (D / 4));
      float top = row_m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, row_m[w][r]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ptx::ex2_approx(row_m[w][r] - base);
        const float4 y = *reinterpret_cast<const float4*>(smem + (w * kRows + r) * kPitch + d);
        sum = fmaf(row_l[w][r], f, sum);
        x.x = fmaf(y.x, f, x.x);
        x.y = fmaf(y.y, f, x.y);
        x.z = fmaf(y.z, f, x.z);
        x.w = fmaf(y.w, f, x.w);
      }
      if (all_keys) {
        const int row = row0 + r;
        if (row < rows_in) {
          const float n = top == -INFINITY ? 0.f : 1.f / sum;
          const int tok = row / p.group;
          T* dst = static_cast<T*>(p.out) + (rq.start + tok) * p.o_token +
                   (kvh * p.group + row - tok * p.group) * p.o_head + d;
          *reinterpret_cast<uint2*>(dst) =
              make_uint2(pack_out<T>(x.x * n, x.y * n), pack_out<T>(x.z * n, x.w * n));
        }
      } else {
        *reinterpret_cast<float4*>(Parts<NT, D>::o(p.ws, slot) + r * D + d) = x;
        if (d == 0)
          Parts<NT, D>::ml(p.ws, 2ll * gridDim.x, slot)[r] = make_float2(top, sum);
      }
    }
    __syncthreads();
    at += c1 - c0;
  }
}

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
  const long long total = count_chunks<NT>(p, part_sum);
  const long long each = chunks_each(total);
  const long long cut = each * (blockIdx.x + 1ll);
  if (threadIdx.x == 0 && cut < total) place = find_place<NT>(p, part_sum, cut);
  __syncthreads();
  // By every CTA, those without work too: this kernel may not end before the
  // one in front of it.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (cut >= total) return;
  const Place pl = place;
  const Request rq = request_at(p, pl.request);
  const Shape sh = shape_of<NT>(p, rq);
  const long long in = cut - pl.before;
  const int unit = static_cast<int>(in / sh.chunks);
  const long long begin = pl.before + static_cast<long long>(unit) * sh.chunks;
  const long long end = begin + sh.chunks;
  if (begin == cut || begin < cut - each) return;  // not cut here, or not for the first time
  const int tiles = sh.units / p.kv_heads;
  const int kvh = unit / tiles;
  const int row0 = (unit - kvh * tiles) * kRows;
  const int rows_in = rq.n * p.group;
  const int parts = static_cast<int>((end - cut + each - 1) / each) + 1;
  const long long slots = 2ll * gridDim.x;

  auto slot_of = [&](int i) { return i == 0 ? 2ll * blockIdx.x + 1 : 2ll * (blockIdx.x + i); };
  for (int r = warp; r < kRows && row0 + r < rows_in; r += 8) {
    float top = -INFINITY;
    for (int i = lane; i < parts; i += 32)
      top = fmaxf(top, Parts<NT, D>::ml(p.ws, slots, slot_of(i))[r].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float x[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) x[j] = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float2 ml = Parts<NT, D>::ml(p.ws, slots, slot_of(i))[r];
      const float f = ptx::ex2_approx(ml.x - base);
      const float* o = Parts<NT, D>::o(p.ws, slot_of(i)) + r * D + lane * (D / 32);
      sum = fmaf(ml.y, f, sum);
      if constexpr (D == 128) {
        const float4 y = *reinterpret_cast<const float4*>(o);
        x[0] = fmaf(y.x, f, x[0]);
        x[1] = fmaf(y.y, f, x[1]);
        x[2] = fmaf(y.z, f, x[2]);
        x[3] = fmaf(y.w, f, x[3]);
      } else {
        const float2 y = *reinterpret_cast<const float2*>(o);
        x[0] = fmaf(y.x, f, x[0]);
        x[1] = fmaf(y.y, f, x[1]);
      }
    }
    const float n = top == -INFINITY ? 0.f : 1.f / sum;
    const int row = row0 + r, tok = row / p.group;
    T* dst = static_cast<T*>(p.out) + (rq.start + tok) * p.o_token +
             (kvh * p.group + row - tok * p.group) * p.o_head + lane * (D / 32);
    if constexpr (D == 128)
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack_out<T>(x[0] * n, x[1] * n), pack_out<T>(x[2] * n, x[3] * n));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack_out<T>(x[0] * n, x[1] * n);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Rows of 8 that a unit holds: as many as the longest request's rows need, up
// to 32; where longer requests go to the tiled kernel, what single tokens need.
int row_tiles(int group, int max_new) {
  const long long rows = static_cast<long long>(group) * max_new;
  const long long want = rows <= 32 ? rows : group;
  return want <= 8 ? 1 : want <= 16 ? 2 : 4;
}

template <int D, int NT>
constexpr size_t smem_bytes() {
  return sizeof(float) * kWarps * 8 * NT * (D + 4) + (NT >= 4 ? NT * (D / 16) * 32 * 8 : 0);
}

template <typename T, int CODE, int D, int NT>
int resident_ctas(int* ctas) {
  static int known[64];  // per device; the same value whoever writes it
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ATTN_ERR_CUDA;
  int n = dev < 64 ? *static_cast<volatile int*>(&known[dev]) : 0;
  if (n == 0) {
    constexpr int smem = static_cast<int>(smem_bytes<D, NT>());
    auto kern = split_kernel<T, CODE, D, NT>;
    int sms = 0, occ = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return ATTN_ERR_RESOURCE;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kThreads, smem) != cudaSuccess)
      return ATTN_ERR_CUDA;
    if (occ < 1) return ATTN_ERR_RESOURCE;
    n = sms * occ;
    if (dev < 64) *static_cast<volatile int*>(&known[dev]) = n;
  }
  *ctas = n;
  return ATTN_OK;
}

constexpr int kMostCtasPerSm = 8;  // bounds the workspace (registers allow fewer)

size_t part_bytes(int D, int nt) { return sizeof(float) * 8 * nt * (D + 2) * 2; }

template <typename T, int CODE, int D, int NT>
int launch(CachedParams p, int max_new, void* ws, unsigned long long ws_bytes, cudaStream_t st) {
  int ctas = 0;
  const int rc = resident_ctas<T, CODE, D, NT>(&ctas);
  if (rc != ATTN_OK) return rc;
  // No more ranges than there can be chunks.
  const long long rows = static_cast<long long>(p.group) * max_new;
  const long long tiles = (rows + 8 * NT - 1) / (8 * NT);
  const long long chunks = p.capacity <= kChunk ? 1 : (p.capacity + kChunk - 1) / kChunk;
  const double most = static_cast<double>(p.batch) * p.kv_heads * tiles * chunks;
  if (most < ctas) ctas = static_cast<int>(most);
  if (ws_bytes < part_bytes(D, NT) * ctas) return ATTN_ERR_SCRATCH_LIMIT;
  p.ws = static_cast<float*>(ws);
  split_kernel<T, CODE, D, NT><<<ctas, kThreads, smem_bytes<D, NT>(), st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return ATTN_ERR_CUDA;
  if (chunks == 1 || ctas == 1) return ATTN_OK;  // no unit can be cut
  // The joining kernel starts while the first still runs (its search of the
  // cuts overlaps) and waits for it before it reads the parts.
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<T, D, NT>, p) == cudaSuccess ? ATTN_OK : ATTN_ERR_CUDA;
}

template <typename T, int CODE, int D>
int launch_nt(const CachedParams& p, int max_new, void* ws, unsigned long long b, cudaStream_t st) {
  switch (row_tiles(p.group, max_new)) {
    case 1: return launch<T, CODE, D, 1>(p, max_new, ws, b, st);
    case 2: return launch<T, CODE, D, 2>(p, max_new, ws, b, st);
    default: return launch<T, CODE, D, 4>(p, max_new, ws, b, st);
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

int launch_split(const CachedParams& p, int D, int dtype, int code, int max_new, void* ws,
                 unsigned long long ws_bytes, cudaStream_t st) {
  return dtype == ATTN_DTYPE_F16 ? launch_code<__half>(p, D, code, max_new, ws, ws_bytes, st)
                                 : launch_code<__nv_bfloat16>(p, D, code, max_new, ws, ws_bytes, st);
}

int split_workspace(int group, int D, int max_new, unsigned long long* bytes) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return ATTN_ERR_CUDA;
  *bytes = part_bytes(D, row_tiles(group, max_new)) * sms * kMostCtasPerSm;
  return ATTN_OK;
}

}  // namespace cache
}  // namespace attnprof
