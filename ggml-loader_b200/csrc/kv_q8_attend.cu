// kv_q8_attend.cu -- attention over the 8-bit cache.
#include <math_constants.h>

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

// One CTA a query row: scores of T keys, then their weighted values; the
// running maximum and sum in float.  ws gets (max, 1 / sum), 0 for a row that adds no weight.
template <int D>
__global__ void __launch_bounds__(T) row_kernel(const AttendParams p)
{
    __shared__ float qs[D], ps[T], red[T / 32];
    const int t = blockIdx.x / p.r, j = blockIdx.x % p.r, h = blockIdx.y, tid = threadIdx.x;
    for (int d = tid; d < D; d += T) qs[d] = query(p, t, h * p.r + j, D, d);
    float m = -CUDART_INF_F, l = 0.0f, o[(D + T - 1) / T] = {};
    __syncthreads();
    for (int64_t base = 0; base < p.n_kv; base += T) {
        const float s = base + tid < p.n_kv ? score<D>(p, qs, h, t, base + tid) : -CUDART_INF_F;
        float x = s;
        for (int k = 16; k; k >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, k));
        if ((tid & 31) == 0) red[tid >> 5] = x;
        __syncthreads();
        float top = m;
        for (int k = 0; k < T / 32; k++) top = fmaxf(top, red[k]);
        const float ref = top == -CUDART_INF_F ? 0.0f : top, f = m == -CUDART_INF_F ? 0.0f : expf(m - ref);
        ps[tid] = s == -CUDART_INF_F ? 0.0f : expf(s - ref);
        __syncthreads();
        l *= f;
#pragma unroll
        for (int k = 0; k < (D + T - 1) / T; k++) o[k] *= f;
        for (int i = 0; i < T && base + i < p.n_kv; i++) {
            const float w = ps[i];
            if (w == 0.0f) continue;
            l += w;
            const int64_t key = base + i;
            const float vs = p.c.v_scale[(int64_t)h * (p.c.rows / kBlock) + key / kBlock];
#pragma unroll
            for (int k = 0; k < (D + T - 1) / T; k++)
                if (tid + k * T < D) o[k] += w * vs * (float)p.c.v[((int64_t)h * p.c.rows + key) * D + tid + k * T];
        }
        m = top;
        __syncthreads();
    }
    const float z = l > 0.0f || l != l ? 1.0f / l : (p.flash ? 0.0f : CUDART_NAN_F);
#pragma unroll
    for (int k = 0; k < (D + T - 1) / T; k++) {
        const int d = tid + k * T;
        if (d >= D) continue;
        const int64_t i = t * p.out_stride + (int64_t)(h * p.r + j) * D + d;
        if (p.out_f16) static_cast<__half *>(p.out)[i] = __float2half_rn(o[k] * z);
        else static_cast<float *>(p.out)[i] = o[k] * z;
    }
    if (tid == 0) {
        const bool adds = l > 0.0f && l < CUDART_INF_F && m < CUDART_INF_F;
        reinterpret_cast<float2 *>(p.ws)[(int64_t)h * p.n_new * p.r + blockIdx.x] =
            adds ? make_float2(m, 1.0f / l) : make_float2(0.0f, 0.0f);
    }
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
        const float2 st = reinterpret_cast<const float2 *>(p.ws)[(int64_t)h * p.n_new * p.r + row];
        if (key < p.n_kv && st.y != 0.0f) sum += expf(score<D>(p, qs, h, t, key) - st.x) * st.y;
    }
    if (key < p.n_kv) p.c.weight[(int64_t)h * p.c.rows + key] += sum;
}

template <int D>
cudaError_t run(const AttendParams &p, cudaStream_t st)
{
    row_kernel<D><<<dim3(p.n_new * p.r, p.c.H), T, 0, st>>>(p);
    if (p.c.weight) weigh_kernel<D><<<dim3((unsigned)((p.n_kv + T - 1) / T), p.c.H), T, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

uint64_t attend_workspace(const AttendParams &p)
{
    return (uint64_t)p.n_new * p.Hq * sizeof(float2);
}

cudaError_t launch_attend(const AttendParams &p, cudaStream_t st)
{
    switch (p.c.D) {
    case 64: return run<64>(p, st);
    case 96: return run<96>(p, st);
    case 128: return run<128>(p, st);
    case 256: return run<256>(p, st);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace q8
}  // namespace kvb
