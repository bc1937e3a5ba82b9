// kv_q8_stage.cuh -- what the tensor-core kernels of the 8-bit cache share:
// codes and queries on their way into swizzled shared memory, bounded waits.
#pragma once

#include "kv_q8.cuh"
#include "kv_sm100.cuh"

namespace kvb {
namespace q8 {

constexpr uint64_t kLimitNs = 1000000000ull;   // bound of every wait: 1 s

__device__ __forceinline__ void give_up(unsigned *error, volatile int *flag, unsigned bit)
{
    if (!*flag) {
        atomicOr(error, bit);
        *flag = 1;
    }
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// four signed codes -> four halves in order (0x6400 | u is the half 1024 + u)
__device__ __forceinline__ uint2 codes_to_half4(uint32_t w)
{
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 hx = __hsub2(*reinterpret_cast<__half2 *>(&x), off), hy = __hsub2(*reinterpret_cast<__half2 *>(&y), off);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&hx), *reinterpret_cast<const uint32_t *>(&hy));
}

// 8 query elements at d as F16
__device__ __forceinline__ uint4 load_q8(const AttendParams &p, int t, int hq, int D, int d)
{
    const int64_t i = t * p.q_stride + (int64_t)hq * D + d;
    uint4 w;
    __half2 *h = reinterpret_cast<__half2 *>(&w);
    if (p.q_f16) {
        const __half *src = static_cast<const __half *>(p.q) + i;
        if (p.q_vec) return *reinterpret_cast<const uint4 *>(src);
#pragma unroll
        for (int k = 0; k < 4; k++) h[k] = __halves2half2(src[2 * k], src[2 * k + 1]);
    } else {
        const float *src = static_cast<const float *>(p.q) + i;
        if (p.q_vec) {
            const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
            h[0] = __floats2half2_rn(a.x, a.y);
            h[1] = __floats2half2_rn(a.z, a.w);
            h[2] = __floats2half2_rn(b.x, b.y);
            h[3] = __floats2half2_rn(b.z, b.w);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) h[k] = __floats2half2_rn(src[2 * k], src[2 * k + 1]);
        }
    }
    return w;
}

__device__ __forceinline__ void sts128(uint32_t at, uint4 v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// 16 codes (chunk c of row r) as F16 in the swizzled layout: box c / 4 (64
// halves a row, 128 bytes), 16-byte chunk j of row r at (j ^ (r & 7)) * 16.
// Half of the lanes store their second chunk first, so 8 lanes fall on
// different banks.
__device__ __forceinline__ void store_codes(uint32_t tile, uint32_t box, int r, int c, uint4 w)
{
    const uint2 a = codes_to_half4(w.x), b = codes_to_half4(w.y), e = codes_to_half4(w.z), f = codes_to_half4(w.w);
    const uint4 lo = make_uint4(a.x, a.y, b.x, b.y), hi = make_uint4(e.x, e.y, f.x, f.y);
    const uint32_t row = tile + (c >> 2) * box + r * 128;
    const int ch = 2 * (c & 3), flip = (c >> 2) & 1;
    sts128(row + (((ch + flip) ^ (r & 7)) << 4), flip ? hi : lo);
    sts128(row + (((ch + 1 - flip) ^ (r & 7)) << 4), flip ? lo : hi);
}

}  // namespace q8
}  // namespace kvb
