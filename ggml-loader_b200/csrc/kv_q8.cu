// kv_q8.cu -- rows into and out of the 8-bit cache: store, load and evict.
//
// A cache block is kBlock rows of one KV head with one power-of-two scale, so
// a value x of the block is its code times 2^e, code = rn(F16(x) / 2^e): the
// division, and a kept row's code moved from exponent a to b (code * 2^(a-b)),
// are exact but for the one rounding to the integer.
#include "kv_internal.h"
#include "kv_q8.cuh"
#include "kv_sm100.cuh"

namespace kvb {
namespace q8 {
namespace {

using sm100::cluster_rank;
using sm100::cluster_sync_all;
using sm100::mapa;
using sm100::pdl_launch_dependents;
using sm100::pdl_wait;

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr)
{
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

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
    pdl_wait();
    pdl_launch_dependents();
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

// U pieces of 8 codes a thread, their loads in flight together; a token's heads
// are neighbours in the output.  Bound by the output's bytes.
template <int D, bool F16, int U>
__global__ void __launch_bounds__(256) load_kernel(const LoadParams p)
{
    const bool is_v = p.k ? blockIdx.y != 0 : true;
    void *out = is_v ? p.v : p.k;
    const int8_t *codes = is_v ? p.c.v : p.c.k;
    const uint32_t *scale = reinterpret_cast<const uint32_t *>(is_v ? p.c.v_scale : p.c.k_scale);
    // (a row has at most 1024 * 32 pieces, a CTA's rows are few: 32 bits from its first row on)
    const uint32_t pieces = p.c.H * (D / 8);
    const int64_t first = (int64_t)blockIdx.x * (256 * U), t0 = first / pieces;
    const uint32_t base = (uint32_t)(first - t0 * pieces);
    uint2 w[U];
    uint32_t s[U];
    int64_t at[U];
    pdl_wait();
    pdl_launch_dependents();
#pragma unroll
    for (int k = 0; k < U; k++) {
        const uint32_t j = base + threadIdx.x + 256 * k, dt = j / pieces, c = j - dt * pieces;
        const int64_t t = t0 + dt, row = p.row0 + t;
        const uint32_t h = c / (D / 8), d = c % (D / 8) * 8;
        at[k] = t < p.n ? t * p.stride + c * 8 : -1;
        if (at[k] >= 0) {
            w[k] = *reinterpret_cast<const uint2 *>(codes + ((int64_t)h * p.c.rows + row) * D + d);
            s[k] = scale[(int64_t)h * (p.c.rows / kBlock) + row / kBlock];
        }
    }
#pragma unroll
    for (int k = 0; k < U; k++) {
        if (at[k] < 0) continue;
        const int e = scale_exp(s[k]);
        const bool bad = (s[k] & 0x7f800000u) == 0x7f800000u;   // a block with values that are not finite
        if constexpr (F16) {
            __half *dst = static_cast<__half *>(out) + at[k];
            __half y[8];
            if (bad) {
                float x[8];
                decode8(w[k], e, x);
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = __float2half_rn(x[j]);
            } else {
                // the codes as halves times 2^e, both exact (2^-24 is the smallest half)
                const __half2 f = __half2half2(__float2half_rn(pow2(e)));
                const uint2 a = codes_to_half4(w[k].x), b = codes_to_half4(w[k].y);
                __half2 *y2 = reinterpret_cast<__half2 *>(y);
                y2[0] = __hmul2(*reinterpret_cast<const __half2 *>(&a.x), f);
                y2[1] = __hmul2(*reinterpret_cast<const __half2 *>(&a.y), f);
                y2[2] = __hmul2(*reinterpret_cast<const __half2 *>(&b.x), f);
                y2[3] = __hmul2(*reinterpret_cast<const __half2 *>(&b.y), f);
            }
            if (p.vec) {
                *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(y);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) dst[j] = y[j];
            }
        } else {
            float *dst = static_cast<float *>(out) + at[k];
            float x[8];
            decode8(w[k], e, x);
            if (p.vec) {
                reinterpret_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
                reinterpret_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) dst[j] = x[j];
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

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kSelCtas = 8;               // a KV head's cluster
constexpr int kSelSlice = 32 * 1024;      // keys a CTA holds in shared memory; with more it reads them each time
constexpr int kSelBins = 4096;

__device__ __forceinline__ void red_cluster_add(uint32_t addr, int v)
{
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// This CTA's counts added to the cluster's in every CTA; few of the counters
// are not zero, so they are sent one by one (all 4096 read from each CTA
// instead: 44 us against 13).  Leaves zeros behind.
template <int BINS>
__device__ __forceinline__ void send_counts(int *s_mine, int *s_all)
{
    for (int i = threadIdx.x; i < BINS; i += kSelThreads) {
        const int x = s_mine[i];
        if (!x) continue;
        s_mine[i] = 0;
        const uint32_t at = sm100::smem_addr(&s_all[i]);
#pragma unroll
        for (int c = 0; c < kSelCtas; c++) red_cluster_add(mapa(at, c), x);
    }
}

// Sum of the warps' totals before `warp` (s_scan: one a warp), and of all.
__device__ __forceinline__ int before_warp(const int *s_scan, int warp, int lane, int &total)
{
    int y = s_scan[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    total = __shfl_sync(0xffffffffu, y, 31);
    const int b = __shfl_sync(0xffffffffu, y, warp ? warp - 1 : 0);
    return warp ? b : 0;
}

// The digit (from the top) in which the want-th largest key lies, by the
// cluster's counts: thread t takes BINS / 1024 digits from the top down.
// `want` becomes what is to be taken within it, `have` what it holds.
template <int BINS>
__device__ __forceinline__ uint32_t find_digit(const int *s_all, int *s_scan, int *s_found, int &want, int &have)
{
    constexpr int M = BINS / kSelThreads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int x[M], total = 0;
#pragma unroll
    for (int j = 0; j < M; j++) total += x[j] = s_all[BINS - 1 - M * tid - j];
    int y = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    if (lane == 31) s_scan[warp] = y;
    __syncthreads();
    int all;
    int before = y - total + before_warp(s_scan, warp, lane, all);
    if (before < want && want <= before + total) {   // one thread
        int digit = BINS - 1 - M * tid;
#pragma unroll
        for (int j = 0; j < M - 1; j++)
            if (before + x[j] < want && digit == BINS - 1 - M * tid - j) {
                before += x[j];
                digit--;
            }
        s_found[0] = digit;
        s_found[1] = want - before;
        s_found[2] = s_all[digit];
    }
    __syncthreads();
    want = s_found[1];
    have = s_found[2];
    return s_found[0];
}

// A cluster a KV head, each CTA a contiguous slice of its candidates: the
// (keep - recent)-th largest key by digits of 12, 10 and 10 bits (histograms in
// shared memory, added up over the cluster; the first digit takes the sign, the
// exponent and 3 bits of the fraction, so that like weights do not meet in one
// counter), then the kept rows in order from each CTA's place on.  The weights
// are read once; what is left are the cluster's barriers, one a digit (32k
// candidates, 8 heads: one CTA a head 140 us, four 8-bit digits 17 us).
__global__ void __cluster_dims__(kSelCtas, 1, 1) __launch_bounds__(kSelThreads) select_kernel(const EvictParams p)
{
    extern __shared__ uint32_t s_dyn[];
    int *s_mine = reinterpret_cast<int *>(s_dyn);        // this CTA's counts
    int *s_all = s_mine + kSelBins;                      // [2][kSelBins] the cluster's, by digit in turn
    uint32_t *s_key = s_dyn + 3 * kSelBins;
    __shared__ int s_scan[2 * kSelWarps];
    __shared__ int s_found[3];
    __shared__ int s_count[2];         // this CTA's keys above the edge, and on it
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)cluster_rank(), h = blockIdx.x / kSelCtas;
    const int cand = (int)(p.n_rows - p.recent), take = (int)(p.keep - p.recent);
    const float *w = p.src.weight + (int64_t)h * p.src.rows;
    int32_t *kept = p.kept + (int64_t)h * p.keep;
    // slices of a multiple of 4 keys
    const int per = (int)(((int64_t)cand + kSelCtas * 4 - 1) / (kSelCtas * 4) * 4);
    const int lo = (int)min((int64_t)cand, (int64_t)rank * per), n = min(per, cand - lo);
    const bool held = per <= kSelSlice;
    for (int i = tid; i < 3 * kSelBins; i += kSelThreads) s_mine[i] = 0;
    cluster_sync_all();   // (counts may come in)
    pdl_wait();
    pdl_launch_dependents();
    for (int64_t j = (int64_t)rank * kSelThreads + tid; j < p.recent; j += kSelCtas * kSelThreads)
        kept[take + j] = cand + (int32_t)j;
    if (take == 0) return;   // (the whole cluster)
    // the first digit with the reading of the weights
#pragma unroll 4
    for (int i = tid; i < n; i += kSelThreads) {
        const uint32_t k = weight_key(w[lo + i]);
        if (held) s_key[i] = k;
        atomicAdd(&s_mine[k >> 20], 1);
    }
    auto key = [&](int i) { return held ? s_key[i] : weight_key(w[lo + i]); };
    int want = take, have;   // still to be taken among the keys with the prefix, and their number
    __syncthreads();
    send_counts<4096>(s_mine, s_all);
    cluster_sync_all();
    uint32_t prefix = find_digit<4096>(s_all, s_scan, s_found, want, have);
    // (find_digit's barrier: the first counts are read; they are zeros again before the last digit's come in)
    s_all[tid] = 0;
    // (where all keys with the prefix are taken -- the cluster's CTAs know the same numbers -- the other digits do not matter)
    int shift = 20;
#pragma unroll 1
    for (int d = 0; d < 2 && want < have; d++) {
        shift -= 10;
        int *all = s_all + (d ? 0 : kSelBins);
        for (int i = tid; i < n; i += kSelThreads) {
            const uint32_t k = key(i);
            if (k >> (shift + 10) == prefix) atomicAdd(&s_mine[(k >> shift) & 1023u], 1);
        }
        __syncthreads();
        send_counts<1024>(s_mine, all);
        cluster_sync_all();
        prefix = prefix << 10 | find_digit<1024>(all, s_scan, s_found, want, have);
    }

    // a thread's keys are neighbours: m of them from m tid on
    const int m = (n + kSelThreads * 4 - 1) / (kSelThreads * 4) * 4, i0 = min(n, m * tid), i1 = min(n, i0 + m);
    int above = 0, on = 0;
    for (int i = i0; i < i1; i++) {
        const uint32_t k = key(i) >> shift;
        above += k > prefix;
        on += k == prefix;
    }
    // exclusive sums over the CTA of both
    int a = above, e = on;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, a, o), z = __shfl_up_sync(0xffffffffu, e, o);
        if (lane >= o) {
            a += y;
            e += z;
        }
    }
    if (lane == 31) {
        s_scan[warp] = a;
        s_scan[kSelWarps + warp] = e;
    }
    __syncthreads();
    int n_above, n_on;
    a += before_warp(s_scan, warp, lane, n_above) - above;
    e += before_warp(s_scan + kSelWarps, warp, lane, n_on) - on;
    if (tid == 0) {
        s_count[0] = n_above;
        s_count[1] = n_on;
    }
    cluster_sync_all();
    {
        // lane c: the counts of CTA c, where it comes before this one
        const uint32_t at = mapa(sm100::smem_addr(s_count), lane & (kSelCtas - 1));
        const bool take_it = lane < rank;
        a += __reduce_add_sync(0xffffffffu, take_it ? ld_cluster_s32(at) : 0);
        e += __reduce_add_sync(0xffffffffu, take_it ? ld_cluster_s32(at + 4) : 0);
    }
    sm100::cluster_arrive();
    // rows before this thread's first: a above the edge and min(e, want) on it
    for (int i = i0; i < i1; i++) {
        const uint32_t k = key(i) >> shift;
        const bool tie = k == prefix;
        if (k > prefix || (tie && e < want)) kept[a + min(e, want)] = lo + i;
        a += k > prefix;
        e += tie;
    }
    sm100::cluster_wait();   // (no CTA leaves while its counts are read)
}

// 16 codes times 2^k, rounded: as halves, whose numbers from 1024 to 2048 are
// the integers, so 1536 + code * 2^k is the rounded code in the low byte (one
// rounding, to even; the factor is exact from 2^-24 on, and 0 below, where every
// code rounds to 0; a code that is not 0 stays below 128, so k < 7 for it).
// bad: kBad codes may be among them.
__device__ __forceinline__ void move_codes(uint4 &x, int k, bool bad)
{
    const __half2 f = __half2half2(__float2half_rn(pow2(min(k, 15)))), one = __half2half2(__ushort_as_half(0x6600));
    uint32_t *w = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint2 y = codes_to_half4(w[i]);
        const __half2 a = __hfma2(*reinterpret_cast<const __half2 *>(&y.x), f, one);
        const __half2 b = __hfma2(*reinterpret_cast<const __half2 *>(&y.y), f, one);
        uint32_t z = __byte_perm(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b), 0x6420);
        if (bad) {
#pragma unroll
            for (int j = 0; j < 32; j += 8)
                if (((w[i] >> j) & 255u) == 0x80u) z = (z & ~(255u << j)) | (0x80u << j);
        }
        w[i] = z;
    }
}

// One block of dst of a KV head a CTA, K and V: a row is D/16 threads, 16 codes
// each of K and of V.  Many small CTAs keep the gathers in flight (32k rows to
// 16k with the selection and the read-back: 45 us; against each other, registers
// for 6 CTAs an SM 44.1 us, for 5 45.7, two blocks a CTA 47, four 51); the codes'
// arithmetic is in halves, two at a time (with conversions to float and back the
// conversions were the bound, 50 us).  A warp a block, all of its rows in
// flight, measured 52 us.
template <int D>
__global__ void __launch_bounds__(kBlock *D / 16, 1536 / (kBlock * D / 16)) gather_kernel(const EvictParams p)
{
    constexpr int T = kBlock * D / 16;
    __shared__ uint32_t part[2][T / 32];
    const int r = threadIdx.x / (D / 16), c = threadIdx.x % (D / 16) * 16;
    const int h = blockIdx.y;
    const int64_t row = (int64_t)blockIdx.x * kBlock + r;
    uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    int e0[2] = {kExpMin, kExpMin};
    pdl_wait();
    pdl_launch_dependents();
    const bool used = row < p.keep;
    if (used) {
        const int64_t from = p.kept[(int64_t)h * p.keep + row], at = ((int64_t)h * p.src.rows + from) * D + c;
        const int64_t sc = (int64_t)h * (p.src.rows / kBlock) + from / kBlock;
        w[0] = *reinterpret_cast<const uint4 *>(p.src.k + at);
        w[1] = *reinterpret_cast<const uint4 *>(p.src.v + at);
        e0[0] = scale_exp(reinterpret_cast<const uint32_t *>(p.src.k_scale)[sc]);
        e0[1] = scale_exp(reinterpret_cast<const uint32_t *>(p.src.v_scale)[sc]);
        if (c == 0 && p.dst.weight) p.dst.weight[(int64_t)h * p.dst.rows + row] = p.src.weight[(int64_t)h * p.src.rows + from];
    }
    // the largest magnitude, code * 2^e: exact in float, whose bits order as it does
#pragma unroll
    for (int v = 0; v < 2; v++) {
        __half2 m2 = __half2half2(__ushort_as_half(0));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint2 y = codes_to_half4(reinterpret_cast<const uint32_t *>(&w[v])[i]);
            m2 = __hmax2(m2, __hmax2(__habs2(*reinterpret_cast<const __half2 *>(&y.x)), __habs2(*reinterpret_cast<const __half2 *>(&y.y))));
        }
        float m = __half2float(__hmax(__low2half(m2), __high2half(m2)));
        const bool bad = m == 128.0f;
        if (bad) {
            const int8_t *q = reinterpret_cast<const int8_t *>(&w[v]);
            int top = 0;
#pragma unroll
            for (int i = 0; i < 16; i++) top = max(top, q[i] == kBad ? 0 : abs((int)q[i]));
            m = (float)top;
        }
        const uint32_t best = __reduce_max_sync(0xffffffffu, __float_as_uint(__fmul_rn(m, pow2(e0[v]))));
        const bool any = __any_sync(0xffffffffu, bad);
        if ((threadIdx.x & 31) == 0) part[v][threadIdx.x >> 5] = best | (any ? 0x80000000u : 0u);
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 2; v++) {
        uint32_t best = 0, flag = 0;
#pragma unroll
        for (int i = 0; i < T / 32; i++) {
            best = max(best, part[v][i] & 0x7fffffffu);
            flag |= part[v][i];
        }
        const bool bad = (flag & 0x80000000u) != 0;
        const int e = block_exp(__uint_as_float(best));
        if (used) {
            if (e != e0[v]) move_codes(w[v], e0[v] - e, bad);
            *reinterpret_cast<uint4 *>((v ? p.dst.v : p.dst.k) + ((int64_t)h * p.dst.rows + row) * D + c) = w[v];
        }
        if (threadIdx.x == 0)
            (v ? p.dst.v_scale : p.dst.k_scale)[(int64_t)h * (p.dst.rows / kBlock) + blockIdx.x] = __uint_as_float(scale_word(e, bad));
    }
}

template <int D>
cudaError_t store_d(const StoreParams &p, dim3 grid, cudaStream_t st)
{
    return p.f16 ? launch_pdl(store_kernel<D, true>, grid, kBlock * D / 8, 0, p, st)
                 : launch_pdl(store_kernel<D, false>, grid, kBlock * D / 8, 0, p, st);
}

template <int D, int U>
cudaError_t load_du(const LoadParams &p, cudaStream_t st)
{
    const int64_t pieces = p.n * p.c.H * (D / 8);   // (2^31 CTAs would be a cache of 2^42 bytes)
    const dim3 grid((unsigned)((pieces + 256 * U - 1) / (256 * U)), p.k && p.v ? 2 : 1);
    return p.f16 ? launch_pdl(load_kernel<D, true, U>, grid, 256, 0, p, st)
                 : launch_pdl(load_kernel<D, false, U>, grid, 256, 0, p, st);
}

template <int D>
cudaError_t load_d(const LoadParams &p, cudaStream_t st)
{
    // four pieces a thread once they leave eight CTAs an SM (16k rows of 8 heads of 128: 1 piece 22 us, 2 18 us, 4
    // 16 us; 9 rows: 1 piece 0.4 us less than 4)
    return p.n * p.c.H * (D / 8) >= (int64_t)kSMs * 8 * 256 * 4 ? load_du<D, 4>(p, st) : load_du<D, 1>(p, st);
}

}  // namespace

cudaError_t launch_store(const StoreParams &p, cudaStream_t st)
{
    const int64_t b0 = p.row0 / kBlock, b1 = (p.row0 + p.n_new + kBlock - 1) / kBlock;
    const dim3 grid((unsigned)(b1 - b0), p.c.H, 2);
    switch (p.c.D) {
    case 64: return store_d<64>(p, grid, st);
    case 96: return store_d<96>(p, grid, st);
    case 128: return store_d<128>(p, grid, st);
    case 256: return store_d<256>(p, grid, st);
    default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_load(const LoadParams &p, cudaStream_t st)
{
    switch (p.c.D) {
    case 64: return load_d<64>(p, st);
    case 96: return load_d<96>(p, st);
    case 128: return load_d<128>(p, st);
    case 256: return load_d<256>(p, st);
    default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_evict(const EvictParams &p, cudaStream_t st)
{
    static Once once;
    cudaError_t e = once.on_device([] {
        return cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * kSelBins + kSelSlice) * 4);
    });
    if (e != cudaSuccess) return e;
    const int64_t cand = p.n_rows - p.recent, per = (cand + kSelCtas * 4 - 1) / (kSelCtas * 4) * 4;
    e = launch_pdl(select_kernel, dim3(p.src.H * kSelCtas), kSelThreads,
                   (size_t)(3 * kSelBins + (per <= kSelSlice ? per : 0)) * 4, p, st);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)((p.keep + kBlock - 1) / kBlock), p.src.H);
    switch (p.src.D) {
    case 64: return launch_pdl(gather_kernel<64>, grid, kBlock * 4, 0, p, st);
    case 96: return launch_pdl(gather_kernel<96>, grid, kBlock * 6, 0, p, st);
    case 128: return launch_pdl(gather_kernel<128>, grid, kBlock * 8, 0, p, st);
    case 256: return launch_pdl(gather_kernel<256>, grid, kBlock * 16, 0, p, st);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace q8
}  // namespace kvb
