// kv_q8_stage.cuh -- what the tensor-core kernels of the 8-bit cache share:
// codes and queries on their way into swizzled shared memory, bounded waits.
#pragma once

#include "kv_q8.cuh"
#include "kv_sm100.cuh"

namespace kvb {
namespace q8 {

__device__ __forceinline__ void give_up(unsigned *error, volatile int *flag, unsigned bit)
{
    if (!*flag) {
        atomicOr(error, bit);
        *flag = 1;
    }
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void sts128(uint32_t at, uint4 v)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// ---- packed F32 pairs
__device__ __forceinline__ uint64_t pk2(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ float2 up2(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// n bytes (a multiple of 16, both addresses 16-byte aligned) into shared memory, completed on `bar`
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t n, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(n), "r"(sm100::smem_addr(bar))
                 : "memory");
}

// 16 bytes into shared memory, or 16 zeros
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void *src, bool have)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}

// 128 query rows as F16 in the swizzled layout, by 128 threads (t); off[row] is
// where a row's elements start, -1 for a row of zeros (shared memory, complete).
// Aligned F16 rows go straight to shared memory (complete after cp_async_wait);
// others through registers, four loads in flight.
template <int D>
__device__ __forceinline__ void stage_queries(const AttendParams &p, uint32_t dst, uint32_t box, const int64_t *off, int t)
{
    constexpr int C = D / 8;
    if (p.q_f16 && p.q_vec) {
        const __half *q = static_cast<const __half *>(p.q);
#pragma unroll 4
        for (int x = t; x < 128 * C; x += 128) {
            const int row = x / C, c = x % C;
            const int64_t at = off[row];
            cp_async_16_or_zero(dst + (c >> 3) * box + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                                q + (at < 0 ? 0 : at + c * 8), at >= 0);
        }
        sm100::cp_async_commit();
    } else {
#pragma unroll 1
        for (int x0 = t; x0 < 128 * C; x0 += 4 * 128) {
            float v[4][8];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int x = x0 + 128 * k;
                const int64_t at = off[x / C], i = at < 0 ? 0 : at + x % C * 8;   // (element 0 exists)
                if (p.q_f16) {
#pragma unroll
                    for (int e = 0; e < 8; e++) v[k][e] = __half2float(static_cast<const __half *>(p.q)[at < 0 ? 0 : i + e]);
                } else if (p.q_vec) {
                    const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + i);
                    const float4 a = src[0], b = src[1];
                    v[k][0] = a.x; v[k][1] = a.y; v[k][2] = a.z; v[k][3] = a.w;
                    v[k][4] = b.x; v[k][5] = b.y; v[k][6] = b.z; v[k][7] = b.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) v[k][e] = static_cast<const float *>(p.q)[at < 0 ? 0 : i + e];
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int x = x0 + 128 * k, row = x / C, c = x % C;
                const bool have = off[row] >= 0;
                uint4 w;
                __half2 *h = reinterpret_cast<__half2 *>(&w);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    h[e] = have ? __floats2half2_rn(v[k][2 * e], v[k][2 * e + 1]) : __half2half2(__ushort_as_half(0));
                sts128(dst + (c >> 3) * box + row * 128 + (((c & 7) ^ (row & 7)) << 4), w);
            }
        }
    }
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
