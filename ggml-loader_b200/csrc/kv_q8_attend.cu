// kv_q8_attend.cu -- attention over the 8-bit cache.
#include <math_constants.h>

#include <algorithm>

#include "kv_internal.h"
#include "kv_q8.cuh"

namespace kvb {
namespace q8 {
namespace {

constexpr int T = 128;

__device__ __forceinline__ float mask_at(const AttendParams &p, int t, int64_t key)
{
    if (!p.mask) return key <= p.n_past + t ? 0.0f : -CUDART_INF_F;
    const int64_t i = t * p.mask_stride + key;
    return p.mask_f16 ? __half2float(static_cast<const __half *>(p.mask)[i]) : static_cast<const float *>(p.mask)[i];
}

template <int D>
__device__ __forceinline__ float score(const AttendParams &p, const float *qs, int h, int t, int64_t key)
{
    const float m = mask_at(p, t, key);
    if (m == -CUDART_INF_F) return m;
    const float ks = p.c.k_scale[(int64_t)h * (p.c.rows / kBlock) + key / kBlock];
    const int8_t *k = p.c.k + ((int64_t)h * p.c.rows + key) * D;
    float s = 0.0f;
    for (int d = 0; d < D; d += 16) {
        const uint4 w = *reinterpret_cast<const uint4 *>(k + d);
        const int8_t *c = reinterpret_cast<const int8_t *>(&w);
#pragma unroll
        for (int i = 0; i < 16; i++) s = fmaf(qs[d + i], (float)c[i], s);
    }
    return fmaf(s, ks * p.scale, m);
}

__device__ __forceinline__ float query(const AttendParams &p, int t, int hq, int D, int d)
{
    const int64_t i = t * p.q_stride + (int64_t)hq * D + d;
    if (p.q_f16) return __half2float(static_cast<const __half *>(p.q)[i]);
    return __half2float(__float2half_rn(static_cast<const float *>(p.q)[i]));
}

// A thread a (KV head, key): the weights of every query row.
template <int D>
__global__ void __launch_bounds__(T) weigh_kernel(const AttendParams p)
{
    __shared__ float qs[D];
    const int h = blockIdx.y;
    const int64_t key = (int64_t)blockIdx.x * T + threadIdx.x;
    float sum = 0.0f;
    for (int row = 0; row < p.n_new * p.r; row++) {
        const int t = row / p.r;
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += T) qs[d] = query(p, t, h * p.r + row % p.r, D, d);
        __syncthreads();
        const float2 st = p.row_stat[(int64_t)h * p.n_new * p.r + row];
        if (key < p.n_kv && st.y != 0.0f)
            sum += (p.mask ? expf(score<D>(p, qs, h, t, key) - st.x) : exp2f(score<D>(p, qs, h, t, key) * 1.4426950408889634f - st.x)) * st.y;
    }
    if (key < p.n_kv) p.c.weight[(int64_t)h * p.c.rows + key] += sum;
}

template <int D>
cudaError_t weigh(const AttendParams &p, cudaStream_t st)
{
    weigh_kernel<D><<<dim3((unsigned)((p.n_kv + T - 1) / T), p.c.H), T, 0, st>>>(p);
    return cudaGetLastError();
}

// The workspace, laid out from `ws` on; returns its bytes.
uint64_t lay_out(AttendParams &p, char *ws)
{
    const uint64_t rows = (uint64_t)p.n_new * p.r;
    const bool chunk = rows > 16;
    if (chunk) chunk_split(p);
    else rows_split(p);
    uint64_t n = 0;
    auto take = [&](uint64_t bytes) {
        char *at = ws + n;
        n += (bytes + 255) / 256 * 256;
        return at;
    };
    // (the most CTAs any call of these heads has, so that larger sizes never need less)
    const uint64_t slots = ((uint64_t)std::max(p.n_vh, kSMs) + p.n_vh) * (chunk ? 128 * p.n_tile : 16);
    p.part = reinterpret_cast<float *>(take(slots * p.c.D * sizeof(float)));
    p.stat = reinterpret_cast<float2 *>(take(slots * sizeof(float2)));
    p.scores = nullptr;
    p.row_stat = nullptr;
    if (p.c.weight && !chunk) p.scores = reinterpret_cast<float *>(take(p.c.H * rows * p.nb * kBlock * sizeof(float)));
    if (p.c.weight && chunk) p.row_stat = reinterpret_cast<float2 *>(take(p.c.H * rows * sizeof(float2)));
    return n;
}

}  // namespace

uint64_t attend_workspace(const AttendParams &p)
{
    AttendParams q = p;
    uint64_t n = lay_out(q, nullptr);
    if ((int64_t)p.n_new * p.r > 16 && p.r <= 16) {   // what the most rows of the other kernel need, so that it suffices for fewer tokens
        q = p;
        q.n_new = 16 / p.r;
        n = std::max(n, lay_out(q, nullptr));
    }
    return n;
}

cudaError_t launch_attend(AttendParams p, void *ws, cudaStream_t st)
{
    lay_out(p, static_cast<char *>(ws));
    const bool chunk = (int64_t)p.n_new * p.r > 16;
    cudaError_t e = chunk ? launch_chunk(p, st) : launch_rows(p, st);
    if (e != cudaSuccess || !p.row_stat) return e;
    switch (p.c.D) {
    case 64: return weigh<64>(p, st);
    case 96: return weigh<96>(p, st);
    case 128: return weigh<128>(p, st);
    default: return weigh<256>(p, st);
    }
}

}  // namespace q8
}  // namespace kvb
