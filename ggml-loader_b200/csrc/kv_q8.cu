// kv_q8.cu -- rows into and out of the 8-bit cache: store, load and evict.
//
// A cache block is kBlock rows of one KV head with one power-of-two scale, so
// a value x of the block is its code times 2^e, code = rn(F16(x) / 2^e): the
// division, and a kept row's code moved from exponent a to b (code * 2^(a-b)),
// are exact but for the one rounding to the integer.
#include "kv_internal.h"
#include "kv_q8.cuh"

namespace kvb {
namespace q8 {
namespace {

__device__ __forceinline__ bool finite(float x)
{
    return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// 8 elements of one row as F16 values, in float
template <bool F16>
__device__ __forceinline__ void load8(const void *base, int64_t at, bool vec, float (&x)[8])
{
    if constexpr (F16) {
        const __half *p = static_cast<const __half *>(base) + at;
        if (vec) {
            const uint4 w = *reinterpret_cast<const uint4 *>(p);
            const __half2 *h = reinterpret_cast<const __half2 *>(&w);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[2 * i] = __low2float(h[i]);
                x[2 * i + 1] = __high2float(h[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __half2float(p[i]);
        }
    } else {
        const float *p = static_cast<const float *>(base) + at;
        if (vec) {
            const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = p[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __half2float(__float2half_rn(x[i]));
    }
}

// 8 codes at scale 2^e; a kBad code becomes a NaN
__device__ __forceinline__ void decode8(uint2 w, int e, float (&x)[8])
{
    const float s = pow2(e);
    const int8_t *c = reinterpret_cast<const int8_t *>(&w);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = c[i] == kBad ? __uint_as_float(0x7fc00000u) : __fmul_rn((float)c[i], s);
}

__device__ __forceinline__ uint2 encode8(const float (&x)[8], int e)
{
    const float inv = pow2(-e);
    uint2 w;
    int8_t *c = reinterpret_cast<int8_t *>(&w);
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = (int8_t)(finite(x[i]) ? to_code(x[i], inv) : kBad);
    return w;
}

// The block's exponent and whether it holds a value that is not finite, from
// every thread's 8 values (zeros where a thread has none).
template <int THREADS>
__device__ __forceinline__ int block_scale(const float (&x)[8], bool &bad)
{
    __shared__ uint32_t part[THREADS / 32];
    float m = 0.0f;
    bool b = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const bool f = finite(x[i]);
        b |= !f;
        m = fmaxf(m, f ? fabsf(x[i]) : 0.0f);
    }
    // magnitudes of finite floats are below 2^31 as integers and order as
    // they do: the top bit carries the flag
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
    const bool any = __any_sync(0xffffffffu, b);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top | (any ? 0x80000000u : 0u);
    __syncthreads();
    uint32_t best = 0, flag = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; i++) {
        best = max(best, part[i] & 0x7fffffffu);
        flag |= part[i];
    }
    bad = (flag & 0x80000000u) != 0;
    return block_exp(__uint_as_float(best));
}

// One CTA a touched block, KV head and K/V: D/8 threads a row, 8 elements each.
// The first block's rows before row0 take part with their present values.
template <int D, bool F16>
__global__ void __launch_bounds__(kBlock *D / 8) store_kernel(const StoreParams p)
{
    constexpr int T = kBlock * D / 8;
    const int r = threadIdx.x / (D / 8), c = threadIdx.x % (D / 8) * 8;
    const int h = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int64_t blk = p.row0 / kBlock + blockIdx.x, row = blk * kBlock + r;
    const bool fresh = row >= p.row0 && row < p.row0 + p.n_new, old = row < p.row0;
    int8_t *codes = (is_v ? p.c.v : p.c.k) + ((int64_t)h * p.c.rows + row) * D + c;
    float *scale = (is_v ? p.c.v_scale : p.c.k_scale) + (int64_t)h * (p.c.rows / kBlock) + blk;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    int e0 = 0;
    if (fresh) {
        const int64_t at = (row - p.row0) * (is_v ? p.v_stride : p.k_stride) + h * D + c;
        load8<F16>(is_v ? p.v : p.k, at, p.vec, x);
    } else if (old) {
        e0 = scale_exp(__float_as_uint(*scale));
        decode8(*reinterpret_cast<const uint2 *>(codes), e0, x);
    }
    bool bad;
    const int e = block_scale<T>(x, bad);   // (its barrier: the old scale is read before it is replaced)
    if (fresh || (old && e != e0)) *reinterpret_cast<uint2 *>(codes) = encode8(x, e);
    if (threadIdx.x == 0) *scale = __uint_as_float(scale_word(e, bad));
    if (fresh && !is_v && c == 0 && p.c.weight) p.c.weight[(int64_t)h * p.c.rows + row] = 0.0f;
}

template <int D, bool F16>
__global__ void __launch_bounds__(256) load_kernel(const LoadParams p)
{
    const int64_t n = p.n * p.c.H * (D / 8), step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += step) {
        const bool is_v = i >= n;
        void *out = is_v ? p.v : p.k;
        if (!out) continue;
        // a token's heads are neighbours in the output
        const int64_t j = is_v ? i - n : i;
        const int c = (int)(j % (D / 8)) * 8;
        const int64_t th = j / (D / 8);
        const int h = (int)(th % p.c.H);
        const int64_t t = th / p.c.H, row = p.row0 + t;
        const int8_t *codes = is_v ? p.c.v : p.c.k;
        const float *scale = is_v ? p.c.v_scale : p.c.k_scale;
        const uint32_t s = __float_as_uint(scale[(int64_t)h * (p.c.rows / kBlock) + row / kBlock]);
        const uint2 w = *reinterpret_cast<const uint2 *>(codes + ((int64_t)h * p.c.rows + row) * D + c);
        float x[8];
        decode8(w, scale_exp(s), x);
        const int64_t at = t * p.stride + h * D + c;
        if constexpr (F16) {
            __half *dst = static_cast<__half *>(out) + at;
            __half y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = __float2half_rn(x[k]);
            if (p.vec) {
                *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(y);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) dst[k] = y[k];
            }
        } else {
            float *dst = static_cast<float *>(out) + at;
            if (p.vec) {
                reinterpret_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
                reinterpret_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) dst[k] = x[k];
            }
        }
    }
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
// weights as integers that order as they do; every NaN above all others, -0 as 0
__device__ __forceinline__ uint32_t weight_key(float w)
{
    if (w != w) return 0xffffffffu;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

constexpr int kSelThreads = 1024;

// One CTA a KV head: the (keep - recent)-th largest key among the candidates by
// four 8-bit digits, then one ordered pass that writes the kept rows.
__global__ void __launch_bounds__(kSelThreads) select_kernel(const EvictParams p)
{
    __shared__ int hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int64_t s_want;
    __shared__ int warp_n[kSelThreads / 32], warp_t[kSelThreads / 32];
    const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *w = p.src.weight + (int64_t)h * p.src.rows;
    int32_t *kept = p.kept + (int64_t)h * p.keep;
    const int64_t cand = p.n_rows - p.recent, take = p.keep - p.recent;
    if (tid == 0) {
        s_prefix = 0;
        s_want = take;   // still to be taken among the keys with the prefix
    }
    __syncthreads();
    for (int shift = 24; shift >= 0 && take > 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
        for (int64_t i = tid; i < cand; i += kSelThreads) {
            const uint32_t key = weight_key(w[i]);
            if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int64_t want = s_want;
            int d = 255;
            while (d > 0 && hist[d] < want) want -= hist[d--];
            s_want = want;
            s_prefix = prefix << 8 | (uint32_t)d;
        }
        __syncthreads();
    }
    const uint32_t edge = s_prefix;
    int64_t ties = take > 0 ? s_want : 0, at = 0;   // rows of key == edge still to take, rows written
    for (int64_t base = 0; base < cand && take > 0; base += kSelThreads) {
        const int64_t i = base + tid;
        const uint32_t key = i < cand ? weight_key(w[i]) : 0;
        const bool tie = i < cand && key == edge;
        const uint32_t tb = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) warp_t[warp] = __popc(tb);
        __syncthreads();
        int before = __popc(tb & ((1u << lane) - 1u)), all = 0;
        for (int k = 0; k < kSelThreads / 32; k++) {
            if (k < warp) before += warp_t[k];
            all += warp_t[k];
        }
        const bool in = i < cand && (key > edge || (tie && before < ties));
        const uint32_t nb = __ballot_sync(0xffffffffu, in);
        if (lane == 0) warp_n[warp] = __popc(nb);
        __syncthreads();
        int pos = __popc(nb & ((1u << lane) - 1u)), n = 0;
        for (int k = 0; k < kSelThreads / 32; k++) {
            if (k < warp) pos += warp_n[k];
            n += warp_n[k];
        }
        if (in) kept[at + pos] = (int32_t)i;
        at += n;
        ties -= min((int64_t)all, ties);
        __syncthreads();
    }
    for (int64_t j = tid; j < p.recent; j += kSelThreads) kept[take + j] = (int32_t)(cand + j);
}

// One CTA a block of dst, KV head and K/V: gathers its rows and stores them.
template <int D>
__global__ void __launch_bounds__(kBlock *D / 8) gather_kernel(const EvictParams p)
{
    constexpr int T = kBlock * D / 8;
    const int r = threadIdx.x / (D / 8), c = threadIdx.x % (D / 8) * 8;
    const int h = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int64_t blk = blockIdx.x, row = blk * kBlock + r;
    const bool used = row < p.keep;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (used) {
        const int64_t from = p.kept[(int64_t)h * p.keep + row];
        const int8_t *codes = is_v ? p.src.v : p.src.k;
        const float *scale = is_v ? p.src.v_scale : p.src.k_scale;
        const uint32_t s = __float_as_uint(scale[(int64_t)h * (p.src.rows / kBlock) + from / kBlock]);
        decode8(*reinterpret_cast<const uint2 *>(codes + ((int64_t)h * p.src.rows + from) * D + c), scale_exp(s), x);
        if (!is_v && c == 0 && p.dst.weight)
            p.dst.weight[(int64_t)h * p.dst.rows + row] = p.src.weight[(int64_t)h * p.src.rows + from];
    }
    bool bad;
    const int e = block_scale<T>(x, bad);
    if (used)
        *reinterpret_cast<uint2 *>((is_v ? p.dst.v : p.dst.k) + ((int64_t)h * p.dst.rows + row) * D + c) = encode8(x, e);
    if (threadIdx.x == 0)
        (is_v ? p.dst.v_scale : p.dst.k_scale)[(int64_t)h * (p.dst.rows / kBlock) + blk] =
            __uint_as_float(scale_word(e, bad));
}

template <int D>
void store_d(const StoreParams &p, dim3 grid, cudaStream_t st)
{
    if (p.f16) store_kernel<D, true><<<grid, kBlock * D / 8, 0, st>>>(p);
    else store_kernel<D, false><<<grid, kBlock * D / 8, 0, st>>>(p);
}

template <int D>
void load_d(const LoadParams &p, unsigned grid, cudaStream_t st)
{
    if (p.f16) load_kernel<D, true><<<grid, 256, 0, st>>>(p);
    else load_kernel<D, false><<<grid, 256, 0, st>>>(p);
}

}  // namespace

cudaError_t launch_store(const StoreParams &p, cudaStream_t st)
{
    const int64_t b0 = p.row0 / kBlock, b1 = (p.row0 + p.n_new + kBlock - 1) / kBlock;
    const dim3 grid((unsigned)(b1 - b0), p.c.H, 2);
    switch (p.c.D) {
    case 64: store_d<64>(p, grid, st); break;
    case 96: store_d<96>(p, grid, st); break;
    case 128: store_d<128>(p, grid, st); break;
    case 256: store_d<256>(p, grid, st); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_load(const LoadParams &p, cudaStream_t st)
{
    const int64_t n = 2 * p.n * p.c.H * (p.c.D / 8);
    const unsigned grid = (unsigned)((n + 255) / 256 < 148 * 64 ? (n + 255) / 256 : 148 * 64);
    switch (p.c.D) {
    case 64: load_d<64>(p, grid, st); break;
    case 96: load_d<96>(p, grid, st); break;
    case 128: load_d<128>(p, grid, st); break;
    case 256: load_d<256>(p, grid, st); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_evict(const EvictParams &p, cudaStream_t st)
{
    select_kernel<<<p.src.H, kSelThreads, 0, st>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)((p.keep + kBlock - 1) / kBlock), p.src.H, 2);
    switch (p.src.D) {
    case 64: gather_kernel<64><<<grid, kBlock * 8, 0, st>>>(p); break;
    case 96: gather_kernel<96><<<grid, kBlock * 12, 0, st>>>(p); break;
    case 128: gather_kernel<128><<<grid, kBlock * 16, 0, st>>>(p); break;
    case 256: gather_kernel<256><<<grid, kBlock * 32, 0, st>>>(p); break;
    default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace q8
}  // namespace kvb
