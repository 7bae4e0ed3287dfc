// attn_cache_append: keys and values of new tokens into a paged cache held in
// 8 bits, with one power-of-two scale for each (block, head) of K and of V.
//
// Per (block, head) that the call writes into, with a = max |x| over its new
// tokens there: e = the least exponent >= -100 with a <= C * 2^e (C = 448 for
// e4m3, 127 for int8); the scale becomes 2^e where the call writes the block's
// first slot, else max(old scale, 2^e).  Where it grew, the codes in front of
// the call's first slot are rounded again to the new scale; then the new
// tokens' codes are round_to_nearest_even(x / scale).  With powers of two that
// is a shift of the exponent: e4m3 codes move exactly unless they fall into
// the subnormals, and every product here is exact in f32 before the one
// rounding to 8 bits.
//
// A number that is not finite cannot be held: its code is 0, and the block's K
// scale becomes NaN for that head (whichever of k and v had it), until the
// block is written from its first slot again.  Scores against such a block are
// NaN for the rows that see it, and masked ones are dropped before they reach
// a sum; a NaN among the values would instead spread to masked rows as 0 * NaN.
//
// Tokens that follow each other into one block (a run) share its scale, so the
// unit of work is one run and one head; nothing orders two runs, so a call may
// have only one for a block.  A CTA of 2 to 8 warps looks at `chunk`
// consecutive tokens of one head and takes the runs that begin there: a short
// run (single tokens, drafts) by one warp, so that several go at once, a longer
// one by the whole CTA, which holds it in registers between finding its largest
// number and rounding it: every number is read once, with all loads on their
// way at the same time.  Half of each warp works on K and half on V, so that
// both can see whether the other met a number that is not finite.
// It reads 2 bytes and writes 1 per element, plus 8 bytes a run and head; long
// prompts are bound by that traffic, single tokens by latency.
#include "cache.cuh"

namespace attnprof {
namespace cache {
namespace {


struct AppendParams {
  const void *k, *v;
  const int* slots;
  uint8_t *kc, *vc;
  float *ks, *vs;
  long long k_token, k_head, v_token, v_head;  // strides in elements
  int tokens, heads, num_slots, shift, chunk;
};

template <typename T>
struct Bits;
template <>
struct Bits<__half> {
  static constexpr uint32_t kInf = 0x7c00u;
  static __device__ __forceinline__ float2 to_float2(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
  }
  static __device__ __forceinline__ float to_float(uint32_t b) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
  }
};
template <>
struct Bits<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80u;
  static __device__ __forceinline__ float2 to_float2(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ float to_float(uint32_t b) { return __uint_as_float(b << 16); }
};

// Both halves of a word: those that are not finite become 0.
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  return w & ~__vcmpgeu2(w & 0x7fff7fffu, Bits<T>::kInf * 0x10001u);
}

// The least e >= kLeastExponent with a <= C * 2^e (a >= 0, finite).
template <int CODE>
__device__ __forceinline__ int exponent_for(float a) {
  const int bits = __float_as_int(a);
  const int e2 = (bits >> 23) - 127;  // a = 1.m * 2^e2 (a subnormal a ends at the bound)
  const int m = bits & 0x7fffff;
  // C = 1.75 * 2^8 and 1.984375 * 2^6
  const int e = CODE == ATTN_CODE_E4M3 ? e2 - 8 + (m > 0x600000 ? 1 : 0)
                                       : e2 - 6 + (m > 0x7e0000 ? 1 : 0);
  return max(e, kLeastExponent);
}

template <typename T, int CODE, int D, int kWarps, int ITERS>
__global__ void __launch_bounds__(32 * kWarps) append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 8;              // lanes on one token's row: 16 bytes each
  constexpr int kRows = 16 / kLanes;         // tokens a half warp takes at once
  constexpr int kShort = 2 * kRows;          // tokens of a run that one warp takes
  __shared__ uint32_t tops[2][kWarps];
  __shared__ uint32_t bads[kWarps];
  begin_behind();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool is_v = lane >= 16;
  const int sub = (lane & 15) / kLanes;      // which of the kRows tokens
  const int part = (lane & 15) % kLanes;     // which 8 elements of the row
  const int bs = 1 << p.shift;
  const int head = static_cast<int>(blockIdx.y);
  const long long begin = static_cast<long long>(blockIdx.x) * p.chunk;
  const long long end = min(begin + p.chunk, static_cast<long long>(p.tokens));

  const T* x = static_cast<const T*>(is_v ? p.v : p.k) + head * (is_v ? p.v_head : p.k_head) +
               8 * part;
  const long long x_token = is_v ? p.v_token : p.k_token;
  uint8_t* codes = is_v ? p.vc : p.kc;
  float* scales = is_v ? p.vs : p.ks;

  // One run: tokens t0 .. t0 + n into slots slot .. slot + n of one block.
  // WHOLE: by all warps together, else by this warp alone.
  auto run = [&](auto whole, long long t0, int n, int slot) {
    constexpr bool WHOLE = decltype(whole)::value;
    constexpr int kIters = WHOLE ? ITERS : kShort / kRows;
    constexpr int kStep = WHOLE ? kRows * kWarps : kRows;
    const int row = (WHOLE ? warp * kRows : 0) + sub;
    const int off = slot & (bs - 1);
    const long long block_head = static_cast<long long>(slot >> p.shift) * p.heads + head;
    float* scale_at = scales + block_head;
    uint8_t* rows = codes + (block_head << p.shift) * D + 8 * part;

    uint4 w[kIters];
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      w[i] = make_uint4(0, 0, 0, 0);
      if (row + i * kStep < n)
        w[i] = __ldcs(reinterpret_cast<const uint4*>(x + (t0 + row + i * kStep) * x_token));
    }
    const float old = off > 0 ? *scale_at : 0.f;
    // Largest |x| of the run, as bits: for finite numbers these order alike,
    // and the others are above them.
    auto largest = [&]() {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kIters; ++i)
        top = __vmaxu2(top, __vmaxu2(__vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu),
                                     __vmaxu2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu)));
      top = max(top & 0xffffu, top >> 16);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(~0u, top, d));
      return top;
    };
    uint32_t top = largest();
    bool any_bad = __any_sync(~0u, top >= Bits<T>::kInf);
    if (any_bad) {
#pragma unroll
      for (int i = 0; i < kIters; ++i) {
        w[i].x = finite_only<T>(w[i].x);
        w[i].y = finite_only<T>(w[i].y);
        w[i].z = finite_only<T>(w[i].z);
        w[i].w = finite_only<T>(w[i].w);
      }
      top = largest();
    }
    if constexpr (WHOLE) {
      if ((lane & 15) == 0) tops[is_v][warp] = top;
      if (lane == 0) bads[warp] = any_bad;
      __syncthreads();  // (every thread has read the old scale, too)
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        top = max(top, tops[is_v][i]);
        any_bad |= bads[i] != 0;
      }
    } else {
      __syncwarp();
    }

    const float want = power_of_two(exponent_for<CODE>(Bits<T>::to_float(top)));
    const bool dead = off > 0 && old != old;  // a NaN scale stays until the block is begun anew
    const float now = (off > 0 && old > want) ? old : want;
    const bool grew = off > 0 && !dead && now > old;
    if ((lane & 15) == 0 && (!WHOLE || warp == 0))
      *scale_at = ((any_bad && !is_v) || dead) ? __int_as_float(0x7fffffff) : now;

    if (grew) {  // codes in front of the run, to the new scale
      const float r = old / now;
      for (int i = row; i < off; i += kStep) {
        uint2* at = reinterpret_cast<uint2*>(rows + static_cast<long long>(i) * D);
        uint2 c = *at;
        uint32_t* u = reinterpret_cast<uint32_t*>(&c);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 a = half2_to_float2(Code<CODE>::half2_lo(u[j]));
          const float2 b = half2_to_float2(Code<CODE>::half2_hi(u[j]));
          u[j] = Code<CODE>::encode4(a.x, a.y, b.x, b.y, r);
        }
        *at = c;
      }
    }
    if ((__float_as_int(now) & 0x7fffff) == 0) {  // a power of two: its reciprocal is exact
      const float inv = 1.f / now;
#pragma unroll
      for (int i = 0; i < kIters; ++i) {
        if (row + i * kStep < n) {
          const float2 a = Bits<T>::to_float2(w[i].x), b = Bits<T>::to_float2(w[i].y);
          const float2 c = Bits<T>::to_float2(w[i].z), d = Bits<T>::to_float2(w[i].w);
          *reinterpret_cast<uint2*>(rows + static_cast<long long>(off + row + i * kStep) * D) =
              make_uint2(Code<CODE>::encode4(a.x, a.y, b.x, b.y, inv),
                         Code<CODE>::encode4(c.x, c.y, d.x, d.y, inv));
        }
      }
    } else {  // a scale that the caller brought
#pragma unroll 1
      for (int i = row; i < n; i += kStep) {
        uint4 v = *reinterpret_cast<const uint4*>(x + (t0 + i) * x_token);
        uint32_t* u = reinterpret_cast<uint32_t*>(&v);
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 a = Bits<T>::to_float2(finite_only<T>(u[j]));
          f[2 * j] = a.x / now;
          f[2 * j + 1] = a.y / now;
        }
        *reinterpret_cast<uint2*>(rows + static_cast<long long>(off + i) * D) =
            make_uint2(Code<CODE>::encode4(f[0], f[1], f[2], f[3], 1.f),
                       Code<CODE>::encode4(f[4], f[5], f[6], f[7], 1.f));
      }
    }
    if constexpr (WHOLE) __syncthreads();  // tops and bads may be written again
  };

  auto slot_at = [&](long long t) {
    const int s = p.slots[t];
    return s >= 0 && s < p.num_slots ? s : -1;
  };

  int short_runs = 0;
  for (long long base = begin; base < end; base += 32) {
    // Tokens base .. base + 31, one a lane: which begin a run (they have a slot
    // into which the token before does not lead), and which go on with one.
    const long long t = base + lane;
    const int mine = t < p.tokens ? slot_at(t) : -1;
    const bool goes_on = mine >= 0 && (mine & (bs - 1)) > 0 && t > 0 && slot_at(t - 1) == mine - 1;
    const unsigned follow = __ballot_sync(~0u, goes_on);
    unsigned starts = __ballot_sync(~0u, mine >= 0 && !goes_on && t < end);
    while (starts != 0) {
      const int s = __ffs(starts) - 1;
      starts &= starts - 1;
      const int slot = __shfl_sync(~0u, mine, s);
      // Tokens that go on behind it, beyond these 32 too.
      const unsigned rest = s == 31 ? 0u : ~(follow >> (s + 1));
      int n = 1 + (s == 31 ? 0 : min(__ffs(rest) - 1, 31 - s));
      if (s + n == 32) {
        const int most = static_cast<int>(
            min(static_cast<long long>(bs - (slot & (bs - 1))), p.tokens - (base + s)));
        while (n < most) {
          const int i = n + lane;
          const unsigned next =
              __ballot_sync(~0u, i < most && p.slots[base + s + i] == slot + i);
          n += next == ~0u ? 32 : __ffs(~next) - 1;
          if (next != ~0u) break;
        }
      }
      if (n > kShort)
        run(std::true_type{}, base + s, n, slot);
      else if (short_runs++ % kWarps == warp)
        run(std::false_type{}, base + s, n, slot);
    }
  }
}

template <typename T, int CODE, int D, int WARPS, int ITERS>
int launch_rounds(const AppendParams& p, cudaStream_t st) {
  const dim3 grid((static_cast<unsigned>(p.tokens) + p.chunk - 1) / p.chunk,
                  static_cast<unsigned>(p.heads));
  return launch_behind(append_kernel<T, CODE, D, WARPS, ITERS>, grid, 32 * WARPS, 0, 0, st, p) ==
                 cudaSuccess
             ? ATTN_OK
             : ATTN_ERR_CUDA;
}

template <typename T, int CODE, int D>
int launch(const AppendParams& p0, cudaStream_t st) {
  AppendParams p = p0;
  // Tokens a CTA looks at: as many as leave some eight CTAs an SM, between one
  // (few tokens: all begin runs) and a block's worth (prompts: one run each).
  const long long per_cta = static_cast<long long>(p.tokens) * p.heads / (148 * 8);
  p.chunk = 1;
  while (2 * p.chunk <= per_cta && p.chunk < (1 << p.shift)) p.chunk *= 2;
  // Rounds of one warp for a whole block; the CTA's warps share them and hold
  // theirs in registers.  On 15,000 tokens of 8 heads of 128: blocks of 16
  // tokens 19.3 us with 2 warps, 21.9 with 4, 37 with 8; of 64 24.4 us with 4,
  // 25.8 with 8, 34 with 16; of 128 28.6 with 8, 32 with 4.
  constexpr int kTokens = 16 / (D / 8);
  switch ((1 << p.shift) / kTokens) {
    case 8: return launch_rounds<T, CODE, D, 2, 4>(p, st);
    case 16: return launch_rounds<T, CODE, D, 2, 8>(p, st);
    case 32: return launch_rounds<T, CODE, D, 4, 8>(p, st);
    case 64: return launch_rounds<T, CODE, D, 4, 16>(p, st);
    default: return launch_rounds<T, CODE, D, 8, 16>(p, st);
  }
}

template <typename T, int CODE>
int launch_d(const AppendParams& p, int D, cudaStream_t st) {
  return D == 64 ? launch<T, CODE, 64>(p, st) : launch<T, CODE, 128>(p, st);
}

template <typename T>
int launch_code(const AppendParams& p, int D, int code, cudaStream_t st) {
  return code == ATTN_CODE_E4M3 ? launch_d<T, ATTN_CODE_E4M3>(p, D, st)
                                : launch_d<T, ATTN_CODE_INT8>(p, D, st);
}

}  // namespace
}  // namespace cache
}  // namespace attnprof

using namespace attnprof::cache;

extern "C" int attn_cache_append(const attn_cache_append_args* args, void* stream) {
  if (!args) return ATTN_ERR_INVALID_ARG;
  const attn_cache_append_args& a = *args;
  const int rc = check_pool(a.num_blocks, a.kv_heads, a.block_size, a.D, a.code);
  if (rc != ATTN_OK) return rc;
  if (!dtype_ok(a.dtype)) return ATTN_ERR_UNSUPPORTED;
  if (a.tokens < 0 || a.kv_heads > 65535) return ATTN_ERR_INVALID_ARG;
  if (a.tokens == 0) return ATTN_OK;
  if (!a.k || !a.v || !a.slots || !a.k_codes || !a.v_codes || !a.k_scale || !a.v_scale)
    return ATTN_ERR_INVALID_ARG;
  if (!aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.k_codes, 16) ||
      !aligned(a.v_codes, 16) || !aligned(a.k_scale, 4) || !aligned(a.v_scale, 4) ||
      !aligned(a.slots, 4) ||
      ((a.k_token_stride | a.k_head_stride | a.v_token_stride | a.v_head_stride) & 7) != 0)
    return ATTN_ERR_MISALIGNED;
  AppendParams p{};
  p.k = a.k;
  p.v = a.v;
  p.slots = a.slots;
  p.kc = static_cast<uint8_t*>(a.k_codes);
  p.vc = static_cast<uint8_t*>(a.v_codes);
  p.ks = a.k_scale;
  p.vs = a.v_scale;
  p.k_token = a.k_token_stride;
  p.k_head = a.k_head_stride;
  p.v_token = a.v_token_stride;
  p.v_head = a.v_head_stride;
  p.tokens = a.tokens;
  p.heads = a.kv_heads;
  p.num_slots = a.num_blocks * a.block_size;
  p.shift = shift_of(a.block_size);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a.dtype == ATTN_DTYPE_F16 ? launch_code<__half>(p, a.D, a.code, st)
                                   : launch_code<__nv_bfloat16>(p, a.D, a.code, st);
}
