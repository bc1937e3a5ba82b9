// kv_q8.cuh -- device helpers of the 8-bit cache's kernels: scale words and
// code conversions.
#pragma once

#include "kv_q8.h"

namespace kvb {
namespace q8 {

constexpr int kBad = -128;   // the code of a value that F16 does not hold as a finite number

// A scale word is the float 2^e, or, for a block with a kBad code, a NaN that
// keeps e + 127 in its low byte (so a rewound block can be stored again).  A
// block in which nothing was stored holds any word, and may be read under a mask
// that hides its keys: its exponent is brought into the format's range, so that
// what is multiplied by the hidden keys' weights of 0 is finite (from other
// exponents a power of two could be infinite), and zeros are rows of zeros.
__device__ __forceinline__ int scale_exp(uint32_t w)
{
    const int e = (int)((w & 0x7f800000u) == 0x7f800000u ? (w & 0xffu) : w >> 23) - 127;
    return max(kExpMin, min(kExpMax, e));
}

__device__ __forceinline__ uint32_t scale_word(int e, bool bad)
{
    return bad ? 0x7fc00000u | (uint32_t)(e + 127) : (uint32_t)(e + 127) << 23;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The smallest e in [kExpMin, kExpMax] at which amax (>= 0, finite) / 2^e
// rounds to at most 127.  amax / 2^(floor(log2 amax) - 6) lies in [64, 128).
__device__ __forceinline__ int block_exp(float amax)
{
    int e = (int)(__float_as_uint(amax) >> 23) - 127 - 6;
    e = max(e, kExpMin);   // (also amax = 0)
    if (__fmul_rn(amax, pow2(-e)) >= 127.5f) e++;
    return min(e, kExpMax);
}

__device__ __forceinline__ int to_code(float y, float inv_scale)
{
    return max(-127, min(127, __float2int_rn(__fmul_rn(y, inv_scale))));
}

// four signed codes -> four halves in order (0x6400 | u is the half 1024 + u)
__device__ __forceinline__ uint2 codes_to_half4(uint32_t w)
{
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 hx = __hsub2(*reinterpret_cast<__half2 *>(&x), off), hy = __hsub2(*reinterpret_cast<__half2 *>(&y), off);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&hx), *reinterpret_cast<const uint32_t *>(&hy));
}

// A launch that may begin its set-up while the kernel before it in the stream
// ends; every kernel launched so waits (pdl_wait) before it touches memory, and
// lets the next one start (pdl_launch_dependents) only then, so that a kernel
// that starts early may rely on all kernels older than the one before it: the
// F16 cache's decode kernel does (kv_attend.cu).
template <class K, class P>
cudaError_t launch_pdl(K kernel, dim3 grid, unsigned block, size_t smem, const P &p, cudaStream_t st, unsigned cluster = 0)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    launched() += e == cudaSuccess;
    return e;
}

}  // namespace q8
}  // namespace kvb
