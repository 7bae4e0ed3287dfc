// The paged cache held in 8 bits: its layout, its two codes and its argument
// checks, shared by the kernels that fill it and the ones that read it.
//
// A pool of num_blocks blocks of block_size tokens (16, 32, 64 or 128):
//   K, V codes   [num_blocks, kv_heads, block_size, D] bytes, D = 64 or 128
//   K, V scales  [num_blocks, kv_heads] f32; a code c stands for c * scale
// so the tokens of one (block, head) lie in one piece of block_size * D bytes
// and share one scale.  Token `pos` of request r lies in block
// tables[r][pos / block_size] at offset pos % block_size.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <type_traits>

#include "attnprof.h"

namespace attnprof {
namespace cache {

constexpr int kLeastExponent = -100;  // of a block's power-of-two scale

inline bool code_ok(int code) { return code == ATTN_CODE_E4M3 || code == ATTN_CODE_INT8; }
inline bool dtype_ok(int dtype) { return dtype == ATTN_DTYPE_F16 || dtype == ATTN_DTYPE_BF16; }
inline bool block_size_ok(int bs) { return bs == 16 || bs == 32 || bs == 64 || bs == 128; }
inline int shift_of(int block_size) {
  return block_size == 16 ? 4 : block_size == 32 ? 5 : block_size == 64 ? 6 : 7;
}
inline bool aligned(const void* p, unsigned n) {
  return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

// Shape checks common to every call on a pool; ATTN_OK or an error.
inline int check_pool(int num_blocks, int kv_heads, int block_size, int D, int code) {
  if (!code_ok(code) || !block_size_ok(block_size) || (D != 64 && D != 128))
    return ATTN_ERR_UNSUPPORTED;
  if (num_blocks <= 0 || kv_heads <= 0) return ATTN_ERR_INVALID_ARG;
  // A slot (block * block_size + offset) is a 32-bit number.
  if (static_cast<long long>(num_blocks) * block_size > INT_MAX) return ATTN_ERR_INVALID_ARG;
  return ATTN_OK;
}

#ifdef __CUDACC__
// ---------------------------------------------------------------------------
// Codes.  E4M3 is the 8-bit float of 4 exponent and 3 mantissa bits (largest
// 448); INT8 is a whole number in [-127, 127].  Both are held exactly by f16.
// ---------------------------------------------------------------------------
template <int CODE>
struct Code;

template <>
struct Code<ATTN_CODE_E4M3> {
  static constexpr float kLargest = 448.f;
  // Two codes (in the low 16 bits) to two f16.
  static __device__ __forceinline__ uint32_t half2_lo(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
        : "=r"(r)
        : "r"(w));
    return r;
  }
  static __device__ __forceinline__ uint32_t half2_hi(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
        : "=r"(r)
        : "r"(w));
    return r;
  }
  // Four numbers in the codes' range, times f, rounded to the nearest code
  // (ties to even), x in the lowest byte.
  static __device__ __forceinline__ uint32_t encode4(float x, float y, float z, float w, float f) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y * f), "f"(x * f));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(w * f), "f"(z * f));
    return lo | (static_cast<uint32_t>(hi) << 16);
  }
};

template <>
struct Code<ATTN_CODE_INT8> {
  static constexpr float kLargest = 127.f;
  // 1024 + u is an f16 whose low byte is u: the bytes with their sign bit
  // flipped are u = code + 128, so code = (1024 + u) - 1152, exact in f16.
  static __device__ __forceinline__ uint32_t biased(uint32_t w, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(w ^ 0x80808080u), "r"(0x64646464u), "r"(sel));
    const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t half2_lo(uint32_t w) { return biased(w, 0x4140); }
  static __device__ __forceinline__ uint32_t half2_hi(uint32_t w) { return biased(w, 0x4342); }
  // Added to 1.5 * 2^23 a number is rounded to a whole one (ties to even), whose
  // low 8 bits are the sum's: one FMA a number, and no conversion.
  static __device__ __forceinline__ uint32_t encode4(float x, float y, float z, float w, float f) {
    constexpr float kWhole = 12582912.f;
    uint32_t lo, hi, r;
    asm("prmt.b32 %0, %1, %2, 0x0040;"
        : "=r"(lo)
        : "r"(__float_as_uint(fmaf(x, f, kWhole))), "r"(__float_as_uint(fmaf(y, f, kWhole))));
    asm("prmt.b32 %0, %1, %2, 0x0040;"
        : "=r"(hi)
        : "r"(__float_as_uint(fmaf(z, f, kWhole))), "r"(__float_as_uint(fmaf(w, f, kWhole))));
    asm("prmt.b32 %0, %1, %2, 0x5410;" : "=r"(r) : "r"(lo), "r"(hi));
    return r;
  }
};

__device__ __forceinline__ float2 half2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// 2^e for e in [-126, 127].
__device__ __forceinline__ float power_of_two(int e) {
  return __int_as_float((e + 127) << 23);
}
#endif  // __CUDACC__

// A launch whose blocks may start while the kernel in front of it in the stream
// ends: every block of `kern` runs begin_behind() before it touches memory.
// cluster: blocks of one, or 0.
template <typename... P, typename... A>
inline cudaError_t launch_behind(void (*kern)(P...), dim3 grid, int threads, size_t smem,
                                 int cluster, cudaStream_t st, const A&... args) {
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Waits for the end of the kernel in front, whose writes are then seen; the
// next one's blocks may start as soon as all blocks of this one are here.
__device__ __forceinline__ void begin_behind() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace cache
}  // namespace attnprof
