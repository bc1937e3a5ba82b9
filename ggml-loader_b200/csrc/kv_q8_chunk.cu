// kv_q8_chunk.cu -- attention over the 8-bit cache for more than 16 query rows
// a KV head (a prompt's chunk), on the 5th-generation tensor cores: tcgen05.mma
// with F32 accumulators in TMEM, operands in shared memory.
//
// The mathematics is kv_q8_rows.cu's: scores t = (q . codes) * ks * scale,
// weights W = e^t 2^ev relative to a running reference of the row, F16, and
//   out = sum W codes_v / sum W 2^-ev,
// so both operands from the cache are its integer codes, exact in F16.  The
// weights are F16 with them (both operands of an MMA have one type), off by up to
// 2^-11 of each, as the F16 cache's kernel rounds them; their low halves, 22 bits
// in all, would be half as many MMAs again on a pipe that is 63 % busy.
// Reference: unmasked rows keep one number M (log2 units of e^t 2^ev), a whole
// one, so that ev - M is exact up to 2^24 and a weight's exponent is rounded
// once.  Past it, a score of 10^7, a row is made NaN: weights would be off by the
// lost exponents or leave F16's range.  (The pair that a mask has is exact there
// too, but costs the loop without a mask a subtraction and an addition a score:
// 512 tokens at 16k 188 us, so 180.)
// With a mask it is a pair (m, me), since a mask of the type's lowest value
// leaves no room next to it for an exponent.
//
// Work: a tile is 128 query rows of one KV head (row = token * r + head of the
// group); a CTA holds two of them (one at head_dim 256), so a sub-tile of 64
// keys staged once feeds both.  A pair is (KV head, block of two tiles), its
// keys the sub-tiles up to the block's last visible key; the pairs' sub-tiles,
// laid end to end, are cut into equal ranges, one CTA each; pairs cut between
// CTAs are joined by fold_kernel.
//
// chunk_kernel (512 threads, registers moved to where they are needed):
//   warps 0-2   issue the MMAs: S_A, S_B (64 columns each, double buffered) and
//               the products P.V; three threads because one thread's issue rate
//               bounds MMAs this narrow
//   warp 3      brings the codes in (bulk copies, 32 KB in flight); owns TMEM
//   warps 4-7   convert them to F16 in the 128-byte-swizzled layout the tensor
//               cores read; also the queries.  (Codes loaded into registers some
//               units ahead: 512 tokens at 16k 262 us, so 175 then: the fence before a
//               tile is handed over waits for every load in flight)
//   warps 8-15  softmax of tile A and tile B, a query row a thread: S from TMEM,
//               weights back as F16 pairs; rescales O when the reference moves;
//               writes a segment's O
// Every wait is inside the CTA and bounded; an expired one sets the error word.
#include <math_constants.h>

#include <algorithm>

#include "kv_internal.h"
#include "kv_q8_stage.cuh"

namespace kvb {
namespace q8 {

__device__ unsigned g_error[2];   // the record of calls on the callers' buffers, and what was taken from it last

namespace {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = 16777216.0f;           // rows without a mask whose reference is larger are NaN
constexpr float kBias = 7.0f, kTop = 15.0f;   // as kv_q8_rows.cu: a new reference's weight is 2^7, it moves past 2^15
constexpr int kThreads = 512;
constexpr int kSub = 64;   // keys of a sub-tile

template <int D>
struct CL {
    static constexpr int NT = D == 256 ? 1 : 2;              // query tiles a CTA holds
    static constexpr int NB = (D + 63) / 64;                 // 64-wide swizzled boxes a row
    static constexpr uint32_t q_tile = NB * 128 * 128;       // bytes
    static constexpr uint32_t box = kSub * 128;              // [64 keys][64 halves]
    static constexpr uint32_t tile = NB * box;               // a K or V sub-tile
    static constexpr int KS = D == 256 ? 2 : D >= 96 ? 4 : 8;
    static constexpr int VS = KS;
    static constexpr uint32_t unit = kSub * D;               // bytes of codes of a sub-tile
    static constexpr int RS = D == 96 ? 5 : 32768 / (int)unit;   // units of codes in flight or waiting: 32 KB
    static constexpr int n_ld = unit / 16 / 128;             // 16-byte pieces a staging thread converts a unit
    static constexpr size_t o_q = 0;
    static constexpr size_t o_k = o_q + NT * (size_t)q_tile;
    static constexpr size_t o_v = o_k + KS * (size_t)tile;
    static constexpr size_t o_raw = o_v + VS * (size_t)tile;
    static constexpr size_t o_off = o_raw + RS * (size_t)unit;   // [NT][128] where the tiles' query rows are
    static constexpr size_t o_bar = o_off + NT * 128 * 8;
    static constexpr int n_bar = 2 + 2 * KS + 2 * VS + 12 + 2 + 3 + 2 * RS;
    static constexpr size_t o_tm = o_bar + n_bar * 8;
    static constexpr size_t bytes = o_tm + 16;
    static_assert(bytes <= 227 * 1024, "shared memory");
};

// ---- the work split --------------------------------------------------------------
__device__ __forceinline__ int subs_of(const AttendParams &p, int b)
{
    const int64_t last = p.mask ? p.n_kv : p.n_past + min((int64_t)p.n_new, (int64_t)(b + 1) * p.tok_blk);
    return (int)((last + kSub - 1) / kSub);
}

// The axis that is cut: of each pair p.gap units, what its beginning costs in
// sub-tiles, then its sub-tiles.
__device__ __forceinline__ int64_t axis_head(const AttendParams &p) { return p.subs + (int64_t)p.n_blk * p.gap; }

__device__ __forceinline__ int64_t pair_start(const AttendParams &p, int pair)
{
    const int b = pair % p.n_blk;
    int64_t x = (int64_t)(pair / p.n_blk) * axis_head(p);
    for (int i = 0; i < b; i++) x += subs_of(p, i) + p.gap;
    return x;
}

__device__ __forceinline__ int64_t cta_begin(const AttendParams &p, int c)
{
    return (int64_t)c * (p.c.H * axis_head(p)) / p.n_cta;
}

// A walk over a CTA's sub-tiles: pair, sub-tile t of [t0, t1) of its n.
struct Walk {
    int pair, t0, t, t1, n;
    int64_t at, end;   // axis: where the pair's sub-tile 0 is, the CTA's end
    __device__ __forceinline__ void begin(const AttendParams &p, int c)
    {
        const int64_t x = cta_begin(p, c);
        end = cta_begin(p, c + 1);
        const int h = (int)(x / axis_head(p));
        int64_t rem = x - (int64_t)h * axis_head(p);
        int b = 0;
        for (; b < p.n_blk - 1; b++) {
            const int k = subs_of(p, b) + p.gap;
            if (rem < k) break;
            rem -= k;
        }
        pair = h * p.n_blk + b;
        at = x - rem + p.gap;
        t0 = t = (int)max((int64_t)0, rem - p.gap);
        span(p);
    }
    __device__ __forceinline__ void span(const AttendParams &p)
    {
        n = subs_of(p, pair % p.n_blk);
        t1 = (int)min((int64_t)n, end - at);   // (below t0: none of this pair's)
    }
    __device__ __forceinline__ bool more() const { return t0 < t1; }   // (an axis that ends in a gap: no pair after it)
    __device__ __forceinline__ void next_pair(const AttendParams &p)
    {
        pair++;
        t0 = t = 0;
        at += n + p.gap;
        t1 = 0;
        if (at < end) span(p);
    }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == n; }
};

// query tiles of block b that hold rows
__device__ __forceinline__ int tiles_of(const AttendParams &p, int b)
{
    return p.n_tile == 2 && b * p.tok_blk + p.tok_tile < p.n_new ? 2 : 1;
}

template <int N>
__device__ __forceinline__ void regs_inc()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ float max32(const uint32_t *v)
{
    float m[4];
#pragma unroll
    for (int a = 0; a < 4; a++) m[a] = fmaxf(__uint_as_float(v[a]), __uint_as_float(v[4 + a]));
#pragma unroll
    for (int e = 8; e < 32; e += 8)
#pragma unroll
        for (int a = 0; a < 4; a++) m[a] = max3(m[a], __uint_as_float(v[e + a]), __uint_as_float(v[e + 4 + a]));
    return max3(m[0], m[1], fmaxf(m[2], m[3]));
}

__device__ __forceinline__ bool bad_scale(uint32_t w) { return (w & 0x7f800000u) == 0x7f800000u; }

// v[e] = v[e] * scale of its block + mask (natural units); a key masked with -inf stays out whatever v holds
__device__ __forceinline__ void add_mask(const AttendParams &p, int tok, int64_t kb, int nvis, float sc0, float sc1,
                                         uint32_t (&v)[64])
{
    const int64_t base = (int64_t)tok * p.mask_stride + kb;
#pragma unroll 1
    for (int q = 0; q < 4; q++) {
        // (at clamped places, so that the loads are in flight together: 22 tokens over 44k keys 170 us; each under its
        // condition they went one after the other, 257 us)
        uint32_t raw[16];
        const int last = (int)min((int64_t)kSub, p.n_kv - kb) - 1;
        if (p.mask_f16) {
#pragma unroll
            for (int e = 0; e < 16; e++) raw[e] = static_cast<const unsigned short *>(p.mask)[base + min(16 * q + e, last)];
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) raw[e] = static_cast<const uint32_t *>(p.mask)[base + min(16 * q + e, last)];
        }
        float m[16];
#pragma unroll
        for (int e = 0; e < 16; e++)
            m[e] = 16 * q + e >= nvis ? -CUDART_INF_F
                   : p.mask_f16 ? __half2float(__ushort_as_half((unsigned short)raw[e])) : __uint_as_float(raw[e]);
        const float sc = q < 2 ? sc0 : sc1;
#pragma unroll
        for (int qq = 0; qq < 4; qq++) {
            if (qq != q) continue;
#pragma unroll
            for (int e = 0; e < 16; e++)
                v[16 * qq + e] = __float_as_uint(m[e] == -CUDART_INF_F ? m[e] : __fmaf_rn(__uint_as_float(v[16 * qq + e]), sc, m[e]));
        }
    }
}

__device__ __forceinline__ void store_out4(const AttendParams &p, int64_t i, float4 x)
{
    if (p.out_f16) {
        __half *dst = static_cast<__half *>(p.out) + i;
        const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
        if (p.out_vec) {
            *reinterpret_cast<uint2 *>(dst) =
                make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
        } else {
            dst[0] = __low2half(a);
            dst[1] = __high2half(a);
            dst[2] = __low2half(b);
            dst[3] = __high2half(b);
        }
    } else {
        float *dst = static_cast<float *>(p.out) + i;
        if (p.out_vec) {
            *reinterpret_cast<float4 *>(dst) = x;
        } else {
            dst[0] = x.x;
            dst[1] = x.y;
            dst[2] = x.z;
            dst[3] = x.w;
        }
    }
}

__device__ __forceinline__ void st_v8(float *p, const float (&x)[8])
{
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                 "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
}

__device__ __forceinline__ void store_out8(const AttendParams &p, int64_t i, const float (&x)[8])
{
    if (p.out_f16 && p.out_vec) {
        uint4 w;
        __half2 *h = reinterpret_cast<__half2 *>(&w);
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
        *reinterpret_cast<uint4 *>(static_cast<__half *>(p.out) + i) = w;
    } else {
        store_out4(p, i, make_float4(x[0], x[1], x[2], x[3]));
        store_out4(p, i + 4, make_float4(x[4], x[5], x[6], x[7]));
    }
}

__device__ __forceinline__ float inverse_sum(float l, bool flash)
{
    return l == 0.0f ? (flash ? 0.0f : CUDART_NAN_F) : 1.0f / l;
}

// Element d (a multiple of 4) of row `in` of a cut pair's partial output: pieces
// of 8 floats, a piece's rows neighbours, so that a warp's rows fill whole
// sectors both where they are written and where they are read.
template <int D>
__device__ __forceinline__ int64_t part_at(int64_t block, int in, int d)
{
    constexpr int rows = 128 * CL<D>::NT;
    return ((block * (D / 8) + (d >> 3)) * rows + in) * 8 + (d & 7);
}

// what the weights' pass reads of a row: weight = 2^((t - m) * unit) * y
__device__ __forceinline__ float2 row_stat_of(float m, float l)
{
    return l > 0.0f && l < CUDART_INF_F && m < CUDART_INF_F ? make_float2(m, 1.0f / l) : make_float2(0.0f, 0.0f);
}

template <int D, bool MASKED>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const AttendParams p)
{
    using L = CL<D>;
    constexpr int KS = L::KS, VS = L::VS;
    constexpr uint32_t kTmO = 256;   // TMEM column of O_A (O_B at + D); S buffers: g * 128 + {0, 64}
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + L::o_bar);
    uint64_t *q_full = bar, *q_empty = bar + 1;
    uint64_t *k_full = bar + 2, *k_empty = k_full + KS;
    uint64_t *v_full = k_empty + KS, *v_empty = v_full + VS;
    uint64_t *s_full = v_empty + VS, *p_full = s_full + 4, *o_ready = p_full + 4;   // [tile][buffer]
    uint64_t *o_full = o_ready + 4, *o_empty = o_full + 1, *drain = o_empty + 1;
    uint64_t *raw_full = drain + 3, *raw_empty = raw_full + L::RS;
    uint32_t *tm_slot = reinterpret_cast<uint32_t *>(smem + L::o_tm);
    volatile int *flag = reinterpret_cast<volatile int *>(smem + L::o_tm + 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;

    if (tid == 0) {
        for (int i = 0; i < L::n_bar; i++) {
            const uint64_t *b = &bar[i];
            const bool staged = b == q_full || (b >= k_full && b < k_full + KS) || (b >= v_full && b < v_full + VS) ||
                                b >= raw_empty;   // the four staging warps
            const bool both = b == q_empty || (b >= k_empty && b < k_empty + KS);   // both S issuers
            const bool stays_away = p.inject == 1 && b == raw_full + 1;   // test hook: one arrival too many is waited for
            mbar_init(&bar[i], (staged || (b >= p_full && b < p_full + 4) ? 4 : b == o_empty ? 8 : both ? 2 : 1) + stays_away);
        }
        *flag = 0;
        fence_mbar_init();
    }
    if (warp == 3) {
        tmem_alloc(tm_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tm_slot;
    Walk w;
    w.begin(p, cta);
    pdl_wait();
    pdl_launch_dependents();

    if (warp < 4) {
        regs_dec<96>();
        if (lane == 0 && warp == 3) {
            // a unit's codes lie in one piece: one bulk copy; rows past the cache are left out (their weights are 0)
            const uint32_t raw = smem_addr(smem + L::o_raw);
            int u = 0;
            bool ok = true;
            for (; ok && w.more(); w.next_pair(p)) {
                const int64_t head = (int64_t)(w.pair / p.n_blk) * p.c.rows;
                for (int t = w.t0; ok && t < w.t1; t++) {
                    const int64_t key0 = (int64_t)t * kSub;
                    const uint32_t n = (uint32_t)min((int64_t)kSub, p.c.rows - key0) * D;
#pragma unroll
                    for (int v = 0; v < 2; v++, u++) {
                        const int s = u % L::RS;
                        if (u >= L::RS && !mbar_wait_ab(&raw_empty[s], (u / L::RS - 1) & 1, p.limit_ns, flag)) {
                            give_up(p.error, flag, 2u);
                            ok = false;
                            break;
                        }
                        mbar_arrive_expect_tx(&raw_full[s], n);
                        bulk_load(raw + s * L::unit, (v ? p.c.v : p.c.k) + (head + key0) * D, n, &raw_full[s]);
                    }
                }
            }
            // none may land after the CTA has gone
            for (int x = u > L::RS ? u - L::RS : 0; x < u; x++) mbar_wait(&raw_full[x % L::RS], (x / L::RS) & 1, p.limit_ns);
        } else if (lane == 0) {
            constexpr uint32_t idS = idesc_f16_f32(128, kSub, false), idO = idesc_f16_f32(128, D, true);
            const uint32_t sq = smem_addr(smem + L::o_q), sk = smem_addr(smem + L::o_k), sv = smem_addr(smem + L::o_v);
            auto wait = [&](uint64_t *b, uint32_t par) {
                if (mbar_wait_ab(b, par, p.limit_ns, flag)) return true;
                give_up(p.error, flag, 1u);
                return false;
            };
            int i = 0;   // sub-tiles of the CTA so far
            bool ok = true;
            if (warp < 2) {
                const int g = warp;
                int n = 0;   // sub-tiles of tile g so far
                for (int seg = 0; ok && w.more(); seg++, w.next_pair(p)) {
                    const bool active = g < tiles_of(p, w.pair % p.n_blk);
                    if (active && !(ok = wait(q_full, seg & 1))) break;
                    for (int t = w.t0; t < w.t1; t++, i++) {
                        const int s = i % KS;
                        if (!(ok = wait(&k_full[s], (i / KS) & 1))) break;
                        if (!active) {   // (in step with the other tile's issuer)
                            mbar_arrive(&k_empty[s]);
                            if (t == w.t1 - 1) mbar_arrive(q_empty);
                            continue;
                        }
                        // the buffer is free once the product that read its weights is done
                        if (n >= 2 && !(ok = wait(&o_ready[g * 2 + (n & 1)], ((n - 2) >> 1) & 1))) break;
                        tc_fence_after();
                        const uint32_t kt = sk + s * L::tile;
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++)
                            umma_ss(tmem + g * 128 + (n & 1) * 64,
                                    sdesc_k_sw128(sq + g * L::q_tile + (kk >> 2) * 16384 + (kk & 3) * 32),
                                    sdesc_k_sw128(kt + (kk >> 2) * L::box + (kk & 3) * 32), idS, kk > 0);
                        umma_commit(&s_full[g * 2 + (n & 1)]);
                        umma_commit(&k_empty[s]);
                        if (t == w.t1 - 1) umma_commit(q_empty);
                        n++;
                    }
                }
            } else {
                int n[2] = {0, 0};
                for (int seg = 0; ok && w.more(); seg++, w.next_pair(p)) {
                    const int nt = tiles_of(p, w.pair % p.n_blk);
                    for (int t = w.t0; ok && t < w.t1; t++, i++) {
                        const int s = i % VS;
                        if (!(ok = wait(&v_full[s], (i / VS) & 1))) break;
                        if (t == w.t0 && seg > 0 && !(ok = wait(o_empty, (seg - 1) & 1))) break;
#pragma unroll
                        for (int g = 0; g < L::NT; g++) {
                            if (g >= nt) continue;
                            if (!(ok = wait(&p_full[g * 2 + (n[g] & 1)], (n[g] >> 1) & 1))) break;
                            tc_fence_after();
                            const uint32_t vt = sv + s * L::tile;
#pragma unroll
                            for (int kk = 0; kk < kSub / 16; kk++)   // 16 keys a step: 8 columns of F16 pairs
                                umma_ts(tmem + kTmO + g * D, tmem + g * 128 + (n[g] & 1) * 64 + kk * 8,
                                        sdesc_mn_sw128(vt + kk * 2048, L::box), idO, !(t == w.t0 && kk == 0));
                            umma_commit(&o_ready[g * 2 + (n[g] & 1)]);
                            n[g]++;
                        }
                        if (!ok) break;
                        umma_commit(&v_empty[s]);
                        if (t == w.t1 - 1) umma_commit(o_full);
                    }
                }
            }
            // every MMA of this thread has completed before TMEM is freed
            umma_commit(&drain[warp]);
            mbar_wait(&drain[warp], 0, p.limit_ns);
        }
    } else if (warp < 8) {
        regs_dec<80>();
        const int st = tid - 128;
        auto wait = [&](uint64_t *b, uint32_t par) {
            // (one answer for the warp: its lanes arrive together)
            const bool got = mbar_wait_ab(b, par, p.limit_ns, flag);
            if (!__all_sync(0xffffffffu, got)) {
                give_up(p.error, flag, 2u);
                return false;
            }
            return true;
        };
        int64_t *off = reinterpret_cast<int64_t *>(smem + L::o_off);
        int i = 0, u = 0;   // sub-tiles and units so far
        bool ok = true;
        // the next unit, as F16 into `tile` once `empty` (phase par) says it is free
        auto convert = [&](unsigned char *tile, uint64_t *full, uint64_t *empty, bool used, uint32_t par) {
            const int s = u % L::RS;
            if (!wait(&raw_full[s], (u / L::RS) & 1)) return false;
            u++;
            constexpr int N = L::n_ld > 4 ? 4 : L::n_ld;   // pieces at a time (8: registers spilled)
            uint4 c[N];
            const uint4 *src = reinterpret_cast<const uint4 *>(smem + L::o_raw + s * L::unit);
#pragma unroll
            for (int j = 0; j < N; j++) c[j] = src[st + 128 * j];
            if (used && !wait(empty, par)) return false;
#pragma unroll
            for (int j0 = 0; j0 < L::n_ld; j0 += N) {
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const int x = st + 128 * (j0 + j);
                    store_codes(smem_addr(tile), L::box, x / (D / 16), x % (D / 16), c[j]);
                    if (j0 + N < L::n_ld) c[j] = src[x + 128 * N];
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(full);
                mbar_arrive(&raw_empty[s]);
            }
            return true;
        };
        for (int seg = 0; w.more(); seg++, w.next_pair(p)) {
            const int h = w.pair / p.n_blk, b = w.pair % p.n_blk, nt = tiles_of(p, b);
            if (seg > 0 && ok) ok = wait(q_empty, (seg - 1) & 1);
            // the tiles before have been staged; a warp that gave up comes here too, and all four leave together
            if (named_sync_or(1, 128, !ok)) break;
            const int tk = st / p.r, in = st - tk * p.r;
#pragma unroll
            for (int g = 0; g < L::NT; g++) {
                const int tok = b * p.tok_blk + g * p.tok_tile + tk;
                off[g * 128 + st] = tk < p.tok_tile && tok < p.n_new ? tok * p.q_stride + (int64_t)(h * p.r + in) * D : -1;
            }
            named_sync(1, 128);
            for (int g = 0; g < nt; g++) stage_queries<D>(p, smem_addr(smem + L::o_q) + g * L::q_tile, 16384, off + g * 128, st);
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            for (int t = w.t0; t < w.t1; t++, i++) {   // (a warp that gives up here goes on to the next segment's barrier)
                const int ks = i % KS, vs = i % VS;
                if (!(ok = convert(smem + L::o_k + ks * L::tile, &k_full[ks], &k_empty[ks], i >= KS, (i / KS - 1) & 1))) break;
                if (!(ok = convert(smem + L::o_v + vs * L::tile, &v_full[vs], &v_empty[vs], i >= VS, (i / VS - 1) & 1))) break;
            }
        }
    } else {
        regs_inc<168>();
        const int g = (warp - 8) >> 2, q4 = warp & 3;
        const int row = q4 * 32 + lane;   // of the tile
        const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
        const uint32_t tS = tmem + lanes + g * 128, tO = tmem + lanes + kTmO + g * D;
        const int tok_in = row / p.r, hd = row - tok_in * p.r;
        auto wait = [&](uint64_t *b, uint32_t par) {
            if (mbar_wait_ab(b, par, p.limit_ns, flag)) return true;
            give_up(p.error, flag, 4u);
            return false;
        };
        const int64_t n_sc = p.c.rows / kBlock;
        int n = 0;
        bool ok = true;
        for (int seg = 0; ok && w.more(); seg++, w.next_pair(p)) {
            const int h = w.pair / p.n_blk, b = w.pair % p.n_blk;
            if (g >= tiles_of(p, b)) {   // no rows in this tile: keep step with the other one
                ok = __all_sync(0xffffffffu, wait(o_full, seg & 1));
                if (ok && lane == 0) mbar_arrive(o_empty);
                continue;
            }
            const int tok = b * p.tok_blk + g * p.tok_tile + tok_in;
            const bool valid = tok_in < p.tok_tile && tok < p.n_new;
            const int64_t lim = !valid ? -1 : MASKED ? p.n_kv - 1 : p.n_past + tok;   // the last key it may see
            const uint32_t *ksc = reinterpret_cast<const uint32_t *>(p.c.k_scale) + h * n_sc;
            const uint32_t *vsc = reinterpret_cast<const uint32_t *>(p.c.v_scale) + h * n_sc;
            float m = -CUDART_INF_F, me = 0.0f, l = 0.0f, bad = 0.0f;
            // a sub-tile's scale words, one sub-tile ahead; a block behind the keys holds anything: the last block's stand for its own
            uint32_t kw[2], vw[2];
            const int64_t last_blk = (p.n_kv - 1) / kBlock;
            auto scales = [&](int t) {
                const int64_t i = min(2 * (int64_t)t, last_blk), j = min(2 * (int64_t)t + 1, last_blk);
                kw[0] = ksc[i];
                kw[1] = ksc[j];
                vw[0] = vsc[i];
                vw[1] = vsc[j];
            };
            scales(w.t0);
            const int n0 = n;
            for (int t = w.t0; t < w.t1; t++, n++) {
                const int bf = n & 1;
                const uint32_t k0 = kw[0], k1 = kw[1], v0 = vw[0], v1 = vw[1];
                if (t + 1 < w.t1) scales(t + 1);
                if (!(ok = __all_sync(0xffffffffu, wait(&s_full[g * 2 + bf], (n >> 1) & 1)))) break;
                tc_fence_after();
                uint32_t v[64];
                tmem_ld32(tS + bf * 64, *reinterpret_cast<uint32_t(*)[32]>(v));
                tmem_ld32(tS + bf * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
                tmem_wait_ld();
                const int64_t kb = (int64_t)t * kSub;
                const int nvis = (int)max((int64_t)0, min((int64_t)kSub, lim - kb + 1));
                const bool k_bad = bad_scale(k0) || bad_scale(k1);
                if (k_bad) {   // visible keys of such a block are NaN
#pragma unroll
                    for (int e = 0; e < 64; e++)
                        if (bad_scale(e < 32 ? k0 : k1)) v[e] = 0x7fc00000u;
                }
                if (!MASKED && !__all_sync(0xffffffffu, nvis == 64)) {
#pragma unroll
                    for (int e = 0; e < 64; e++)
                        if (e >= nvis) v[e] = __float_as_uint(-CUDART_INF_F);
                }
                const float ev0 = (float)scale_exp(v0), ev1 = (float)scale_exp(v1);
                float c0 = p.scale * pow2(scale_exp(k0)), c1 = p.scale * pow2(scale_exp(k1));
                float f = 1.0f;
                bool moved = false;
                uint64_t s0 = 0ull, s1 = 0ull;
                if constexpr (MASKED) {
                    add_mask(p, valid ? tok : 0, kb, nvis, c0, c1, v);
                    const float x0 = max32(v), x1 = max32(v + 32);
                    // the block whose top counts for more
                    const bool second = x0 == -CUDART_INF_F || (x1 - x0) * kLog2e + (ev1 - ev0) > 0.0f;
                    const float top = second ? x1 : x0, tev = second ? ev1 : ev0;
                    if (top > -CUDART_INF_F && (m == -CUDART_INF_F || __fmaf_rn(top - m, kLog2e, tev - me) > kTop)) {
                        if (m > -CUDART_INF_F) {
                            f = ex2_approx(__fmaf_rn(m - top, kLog2e, me - (tev - kBias)));
                            moved = true;
                        }
                        m = top;
                        me = tev - kBias;
                    }
                    if ((bad_scale(v0) && x0 > -CUDART_INF_F) || (bad_scale(v1) && x1 > -CUDART_INF_F)) bad = CUDART_NAN_F;
                    const float mm = m == -CUDART_INF_F ? 0.0f : m;
                    // (its own loop: the difference is taken before the exponent is added)
                    float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        uint32_t pkd[16];
                        const float up = (u ? ev1 : ev0) - me;
                        float a = 0.0f;
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float y0 = ex2_approx(__fmaf_rn(__uint_as_float(v[u * 32 + 2 * e]) - mm, kLog2e, up));
                            const float y1 = ex2_approx(__fmaf_rn(__uint_as_float(v[u * 32 + 2 * e + 1]) - mm, kLog2e, up));
                            a += y0 + y1;
                            const __half2 h2 = __floats2half2_rn(y0, y1);
                            pkd[e] = *reinterpret_cast<const uint32_t *>(&h2);
                        }
                        if (u) a1 = a;
                        else a0 = a;
                        tmem_st16(tS + bf * 64 + u * 16, pkd);
                    }
                    l = __fmaf_rn(a1, pow2(-(int)ev1), __fmaf_rn(a0, pow2(-(int)ev0), l * f));
                } else {
                    c0 *= kLog2e;
                    c1 *= kLog2e;
                    const float x0 = max32(v), x1 = max32(v + 32);
                    const float z = fmaxf(__fmaf_rn(x0, c0, ev0), __fmaf_rn(x1, c1, ev1));
                    if (z > m + kTop) {   // (never without a visible key: z = -inf)
                        const float to = rintf(z) - kBias;
                        f = ex2_approx(m - to);   // 0 while m = -inf
                        moved = m != -CUDART_INF_F;
                        m = to;
                    }
                    if ((bad_scale(v0) && x0 > -CUDART_INF_F) || (bad_scale(v1) && x1 > -CUDART_INF_F)) bad = CUDART_NAN_F;
                    const float ref = m == -CUDART_INF_F ? 0.0f : m;
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        uint32_t pkd[16];
                        const uint64_t c2 = u ? pk2(c1, c1) : pk2(c0, c0), a2 = u ? pk2(ev1 - ref, ev1 - ref) : pk2(ev0 - ref, ev0 - ref);
                        uint64_t sum = 0ull;
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float2 xy = up2(fma2(pk2(__uint_as_float(v[u * 32 + 2 * e]), __uint_as_float(v[u * 32 + 2 * e + 1])), c2, a2));
                            const float y0 = ex2_approx(xy.x), y1 = ex2_approx(xy.y);
                            sum = add2(sum, pk2(y0, y1));
                            const __half2 h2 = __floats2half2_rn(y0, y1);
                            pkd[e] = *reinterpret_cast<const uint32_t *>(&h2);
                        }
                        if (u) s1 = sum;
                        else s0 = sum;
                        tmem_st16(tS + bf * 64 + u * 16, pkd);
                    }
                    const float2 a0 = up2(s0), a1 = up2(s1);
                    l = __fmaf_rn(a1.x + a1.y, pow2(-(int)ev1), __fmaf_rn(a0.x + a0.y, pow2(-(int)ev0), l * f));
                }
                // O holds the segment's earlier sub-tiles: scaled once the last product into it is done
                if (n > n0 && __any_sync(0xffffffffu, moved)) {
                    if (!(ok = __all_sync(0xffffffffu, wait(&o_ready[g * 2 + ((n - 1) & 1)], ((n - 1) >> 1) & 1)))) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int ch = 0; ch < D / 16; ch++) {
                        uint32_t o[16];
                        tmem_ld16(tO + ch * 16, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st16(tO + ch * 16, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[g * 2 + bf]);
            }
            if (!ok || !(ok = __all_sync(0xffffffffu, wait(o_full, seg & 1)))) break;
            tc_fence_after();
            const bool whole = w.whole();
            const int64_t block = (int64_t)cta + w.pair;   // (CTA, pair) in order: their sum counts them
            const int in = g * 128 + row;
            float scl = 1.0f;
            if constexpr (!MASKED) {   // (m = -inf: no visible key)
                const float far = fabsf(m) >= kFar && m != -CUDART_INF_F ? CUDART_NAN_F : 0.0f;
                l += far;
                bad += far;
            }
            if constexpr (MASKED) {   // both sums relative to e^m alone
                scl = pow2((int)me);
                l *= scl;
            }
            if (whole) scl *= inverse_sum(l, p.flash != 0);
            if (valid) {
                if (!whole) p.stat[block * (128 * L::NT) + in] = make_float2(m, l);
                else if (p.row_stat) p.row_stat[(int64_t)h * p.n_new * p.r + (int64_t)tok * p.r + hd] = row_stat_of(m, l);
            }
            const int64_t dst = (int64_t)tok * p.out_stride + (int64_t)(h * p.r + hd) * D;
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ch++) {
                uint32_t o[32];
                tmem_ld32(tO + ch * 32, o);
                tmem_wait_ld();
                if (!valid) continue;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = __fmaf_rn(__uint_as_float(o[8 * q + e]), scl, bad);
                    if (whole) store_out8(p, dst + ch * 32 + 8 * q, x);
                    else st_v8(p.part + part_at<D>(block, in, ch * 32 + 8 * q), x);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
        if (lane == 0 && p.gave_up) p.gave_up[cta] = *flag;
    }
}

// Joins the pairs cut between CTAs, a warp a query row; row_stat of their rows.
constexpr int kFoldU = 4;

template <int D, bool MASKED, bool WIDE>
__global__ void __launch_bounds__(256) fold_kernel(const AttendParams p)
{
    __shared__ float4 s_o[WIDE ? 8 : 1][D / 4];
    __shared__ float2 s_ml[8];
    constexpr int rows_blk = 128 * CL<D>::NT;
    constexpr float unit = MASKED ? kLog2e : 1.0f;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int rows_cta = WIDE ? 1 : 8;
    const int pair = blockIdx.x / (rows_blk / rows_cta), in = blockIdx.x % (rows_blk / rows_cta) * rows_cta + (WIDE ? 0 : warp);
    const int h = pair / p.n_blk, b = pair % p.n_blk, tk = (in & 127) / p.r, hd = (in & 127) - tk * p.r;
    const int tok = b * p.tok_blk + (in >> 7) * p.tok_tile + tk;
    const int64_t W = p.c.H * axis_head(p), x0 = pair_start(p, pair) + p.gap, x1 = x0 + subs_of(p, b) - 1;
    int c0, c1;
    if ((W + 1) * p.n_cta < ((int64_t)1 << 31)) {   // (a 64-bit division is some hundred instructions)
        c0 = (int)(((uint32_t)(x0 + 1) * (uint32_t)p.n_cta - 1u) / (uint32_t)W);
        c1 = (int)(((uint32_t)(x1 + 1) * (uint32_t)p.n_cta - 1u) / (uint32_t)W);
    } else {
        c0 = (int)(((x0 + 1) * p.n_cta - 1) / W);
        c1 = (int)(((x1 + 1) * p.n_cta - 1) / W);
    }
    pdl_wait();
    pdl_launch_dependents();
    if (c0 == c1 || tk >= p.tok_tile || tok >= p.n_new) return;
    constexpr int V = (D / 4 + 31) / 32;
    float4 x[V];
#pragma unroll
    for (int v = 0; v < V; v++) x[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float M = -CUDART_INF_F, l = 0.0f;
    // kFoldU parts and their (m, l) in flight together
    for (int c = c0 + (WIDE ? warp * kFoldU : 0); c <= c1; c += WIDE ? 8 * kFoldU : kFoldU) {
        float2 s[kFoldU];
        float4 y[kFoldU][V];
#pragma unroll
        for (int u = 0; u < kFoldU; u++) {
            const bool have = c + u <= c1;
            const int64_t block = (int64_t)c + u + pair;
            s[u] = have ? p.stat[block * rows_blk + in] : make_float2(-CUDART_INF_F, 0.0f);
#pragma unroll
            for (int v = 0; v < V; v++) {
                y[u][v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (have && lane + 32 * v < D / 4)
                    y[u][v] = __ldcg(reinterpret_cast<const float4 *>(p.part + part_at<D>(block, in, (lane + 32 * v) * 4)));
            }
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < kFoldU; u++) top = fmaxf(top, s[u].x);
        const float ref = top == -CUDART_INF_F ? 0.0f : top, f0 = ex2_approx((M - ref) * unit);
        M = top;
        l *= f0;
#pragma unroll
        for (int v = 0; v < V; v++) x[v] = make_float4(x[v].x * f0, x[v].y * f0, x[v].z * f0, x[v].w * f0);
#pragma unroll
        for (int u = 0; u < kFoldU; u++) {
            const float f = ex2_approx((s[u].x - ref) * unit);
            l = __fmaf_rn(s[u].y, f, l);
#pragma unroll
            for (int v = 0; v < V; v++) {
                x[v].x = __fmaf_rn(y[u][v].x, f, x[v].x);
                x[v].y = __fmaf_rn(y[u][v].y, f, x[v].y);
                x[v].z = __fmaf_rn(y[u][v].z, f, x[v].z);
                x[v].w = __fmaf_rn(y[u][v].w, f, x[v].w);
            }
        }
    }
    if constexpr (WIDE) {
        // the warps' sums, each relative to its own maximum
#pragma unroll
        for (int v = 0; v < V; v++)
            if (lane + 32 * v < D / 4) s_o[warp][lane + 32 * v] = x[v];
        if (lane == 0) s_ml[warp] = make_float2(M, l);
        __syncthreads();
        if (warp) return;
        M = -CUDART_INF_F;
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) M = fmaxf(M, s_ml[k].x);
        const float ref = M == -CUDART_INF_F ? 0.0f : M;
#pragma unroll
        for (int v = 0; v < V; v++) x[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float f = ex2_approx((s_ml[k].x - ref) * unit);
            l = __fmaf_rn(s_ml[k].y, f, l);
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (lane + 32 * v >= D / 4) continue;
                const float4 y = s_o[k][lane + 32 * v];
                x[v] = make_float4(__fmaf_rn(y.x, f, x[v].x), __fmaf_rn(y.y, f, x[v].y), __fmaf_rn(y.z, f, x[v].z), __fmaf_rn(y.w, f, x[v].w));
            }
        }
    }
    const float z = inverse_sum(l, p.flash != 0);
    const int64_t dst = (int64_t)tok * p.out_stride + (int64_t)(h * p.r + hd) * D;
#pragma unroll
    for (int v = 0; v < V; v++)
        if (lane + 32 * v < D / 4)
            store_out4(p, dst + (lane + 32 * v) * 4, make_float4(x[v].x * z, x[v].y * z, x[v].z * z, x[v].w * z));
    if (lane == 0 && p.row_stat) p.row_stat[(int64_t)h * p.n_new * p.r + (int64_t)tok * p.r + hd] = row_stat_of(M, l);
}

template <int D, bool MASKED>
cudaError_t run(const AttendParams &p, cudaStream_t st)
{
    using L = CL<D>;
    static Once once;
    cudaError_t e = once.on_device([] {
        return cudaFuncSetAttribute(chunk_kernel<D, MASKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::bytes);
    });
    if (e == cudaSuccess) e = launch_pdl(chunk_kernel<D, MASKED>, p.n_cta, kThreads, L::bytes, p, st);
    if (e != cudaSuccess) return e;
    // every pair in one CTA: as many CTAs as pairs of equal length, or one CTA
    if (p.n_cta == 1 || (p.n_blk == 1 && p.c.H % p.n_cta == 0)) return cudaSuccess;
    // pairs of many parts: a CTA a row, its warps share the parts (one head over 21k keys, 148 parts: 98 us with a warp a row)
    if (p.n_cta > 12 * p.n_vh) return launch_pdl(fold_kernel<D, MASKED, true>, (unsigned)p.n_vh * (128 * L::NT), 256, 0, p, st);
    return launch_pdl(fold_kernel<D, MASKED, false>, (unsigned)p.n_vh * (128 * L::NT / 8), 256, 0, p, st);
}

// a record's bits, cleared in the same step: one that another stream's kernel sets meanwhile is not lost
__global__ void take_kernel(unsigned *record) { record[1] = atomicExch(record, 0u); }

}  // namespace

void chunk_split(AttendParams &p)
{
    p.n_tile = p.c.D == 256 ? 1 : 2;
    p.tok_tile = 128 / p.r;
    p.tok_blk = p.n_tile * p.tok_tile;
    p.n_blk = (p.n_new + p.tok_blk - 1) / p.tok_blk;
    p.n_vh = p.c.H * p.n_blk;
    p.subs = 0;
    for (int b = 0; b < p.n_blk; b++) {
        const int64_t last = p.mask ? p.n_kv : p.n_past + std::min<int64_t>(p.n_new, (int64_t)(b + 1) * p.tok_blk);
        p.subs += (last + kSub - 1) / kSub;
    }
    p.n_cta = (int)std::min<int64_t>(kSMs, p.c.H * p.subs);
    // A pair's beginning and end cost a CTA about 8 us, 6 sub-tiles (512 tokens
    // at 4k: CTAs of one pair were done after 50 us, of two after 67); where
    // the ranges are short they stay even, for the sake of more CTAs.
    p.gap = (int)std::min<int64_t>(6, p.c.H * p.subs / p.n_cta / 8);
}

cudaError_t launch_chunk(const AttendParams &p, cudaStream_t st)
{
    switch (p.c.D) {
    case 64: return p.mask ? run<64, true>(p, st) : run<64, false>(p, st);
    case 96: return p.mask ? run<96, true>(p, st) : run<96, false>(p, st);
    case 128: return p.mask ? run<128, true>(p, st) : run<128, false>(p, st);
    case 256: return p.mask ? run<256, true>(p, st) : run<256, false>(p, st);
    default: return cudaErrorInvalidValue;
    }
}

cudaError_t error_word(unsigned **dev)
{
    // (looked up once a device: its address does not change)
    static std::atomic<unsigned *> known[64];
    int id = 0;
    cudaError_t e = cudaGetDevice(&id);
    if (e != cudaSuccess) return e;
    if (id < 64 && (*dev = known[id].load(std::memory_order_relaxed))) return cudaSuccess;
    e = cudaGetSymbolAddress(reinterpret_cast<void **>(dev), g_error);
    if (e == cudaSuccess && id < 64) known[id].store(*dev, std::memory_order_relaxed);
    return e;
}

cudaError_t take_error(unsigned *record, cudaStream_t st, unsigned *word)
{
    take_kernel<<<1, 1, 0, st>>>(record);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpyAsync(word, record + 1, sizeof(unsigned), cudaMemcpyDeviceToHost, st);
    return e == cudaSuccess ? cudaStreamSynchronize(st) : e;
}

}  // namespace q8
}  // namespace kvb
