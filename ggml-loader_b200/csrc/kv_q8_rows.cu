// kv_q8_rows.cu -- attention over the 8-bit cache for up to 16 query rows a KV
// head (a token, a few draft tokens): one pass over the codes.
//
// For a query row, with t_k = (q . c_k) * ks * scale (c_k the codes of key k,
// ks its block's scale, q rounded to F16) and v_k = c'_k * 2^ev:
//   out = sum_k e^(t_k) 2^(ev) c'_k / sum_k e^(t_k).
// Everything in sight of the tensor cores is an integer code or a weight
// W = e^(t - m) 2^(ev - me), F16: a row's reference (m, me) is the score and
// value exponent (less kBias) of the block in which t + ev ln 2 was largest, so
// the largest W lies in [2^7, 2^15] whatever the scales are (a W in F16's
// subnormals is below 2^-21 of it), and the output sums to O * 2^me.  The row's
// sum of e^(t - m) adds W * 2^(me - ev) in float.  With a reference that only
// moves when W would pass 2^15 the accumulators are seldom rescaled.
//
// The tensor cores (mma.sync m16n8k16; tcgen05 has 64 rows at least) are the
// bound next to HBM: with the rows on their 16-wide side and the keys on the
// 8-wide one, half of it empty, their pipe was 82 % busy at 4 rows.  So keys,
// and then dims, are the 16-wide side and 8 rows the 8-wide one: half as many.
//
// A head's blocks are streamed once: warps take blocks of 32 keys in turn, each
// with its own ring of shared memory (cp.async, nothing but warp barriers in
// the loop); partial (m, sum, out) rows of the CTAs of a head are joined in
// their cluster, or by a second kernel launched programmatically.
//
// One token, 8 heads of 128 with 4 query heads each: 131k keys 51 us, 5.2
// TB/s (268 MB; at that length the power limit lowers the clock, and the SMs
// issue an instruction in 54 % of their cycles), 32k keys 17.5 us, of which
// about 7 are the launch, the first loads' latency and the joins.
#include <math_constants.h>

#include <algorithm>

#include "kv_internal.h"
#include "kv_q8.cuh"
#include "kv_sm100.cuh"

namespace kvb {
namespace q8 {
namespace {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxCluster = 8;
constexpr float kBias = 7.0f;    // a new reference's weight is 2^kBias,
constexpr float kTop = 15.0f;    // and it moves where a weight would pass 2^kTop

// NG: groups of 8 query rows.  DUP (up to 4 rows): columns 4-7 of the group
// repeat rows 0-3 and carry the low halves of their weights, W - F16(W), so the
// weights enter with 22 bits at no cost; otherwise in F16 (11 bits, off by up to
// 2^-11 of each, as the F16 cache's kernels round them and as an F16 output is
// rounded once more; their low halves would be as many products again).
template <int D, int NG, int W_>
struct Rows {
    static constexpr int W = W_;                                     // warps
    static constexpr int E = 219 * 1024 / (W * kBlock * (D + 16));   // tiles in a warp's ring
    static constexpr int pitch = D + 16;                             // bytes a row: 8 rows fall on different banks
    static constexpr int tile = kBlock * pitch;                      // K or V of a block
    static constexpr int ring = E * tile;                            // a warp's
    static constexpr int NR = 8 * NG;
    static constexpr int smem = W * ring;                            // (at the end also the W warps' output rows, and their sum)
    static constexpr int nk = D / 16;                                // 16-wide steps over D
    static constexpr bool q_regs = D <= 128 || NG == 1;              // the queries stay in registers, else in shared memory
    static_assert(smem >= (W + 1) * NR * D * 4 && smem <= 225 * 1024, "shared memory");
};

// two F16 pairs (codes 0, 1 | 2, 3 or 0, 2 | 1, 3) of four signed codes: 0x6400
// | u is the half 1024 + u, u = code + 128
template <bool BY_TWO>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &a, uint32_t &b)
{
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
    uint32_t x = __byte_perm(u, 0x64646464u, BY_TWO ? 0x4240 : 0x4140);
    uint32_t y = __byte_perm(u, 0x64646464u, BY_TWO ? 0x4341 : 0x4342);
    const __half2 hx = __hsub2(*reinterpret_cast<__half2 *>(&x), off), hy = __hsub2(*reinterpret_cast<__half2 *>(&y), off);
    a = *reinterpret_cast<const uint32_t *>(&hx);
    b = *reinterpret_cast<const uint32_t *>(&hy);
}

// 8x8 halves, a row a 4 lanes, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 4 query elements from element i on, as two F16 pairs
__device__ __forceinline__ uint2 load_q4(const AttendParams &p, int64_t i)
{
    __half x[4];
    if (p.q_f16) {
        if (p.q_vec) return *reinterpret_cast<const uint2 *>(static_cast<const __half *>(p.q) + i);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = static_cast<const __half *>(p.q)[i + k];
    } else if (p.q_vec) {
        const float4 v = *reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + i);
        x[0] = __float2half_rn(v.x);
        x[1] = __float2half_rn(v.y);
        x[2] = __float2half_rn(v.z);
        x[3] = __float2half_rn(v.w);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = __float2half_rn(static_cast<const float *>(p.q)[i + k]);
    }
    return make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
}

__device__ __forceinline__ void l2_prefetch_bulk(const void *p, uint32_t bytes)
{
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

__device__ __forceinline__ float mask_value(const AttendParams &p, int t, int64_t key)
{
    const int64_t i = t * p.mask_stride + key;
    return p.mask_f16 ? __half2float(static_cast<const __half *>(p.mask)[i]) : static_cast<const float *>(p.mask)[i];
}

__device__ __forceinline__ void store_out(const AttendParams &p, int64_t i, float x)
{
    if (p.out_f16) static_cast<__half *>(p.out)[i] = __float2half_rn(x);
    else static_cast<float *>(p.out)[i] = x;
}

__device__ __forceinline__ int64_t out_at(const AttendParams &p, int h, int row, int D)
{
    const int t = row / p.r;
    return t * p.out_stride + (int64_t)(h * p.r + row - t * p.r) * D;
}

// x * z at four elements from i on
__device__ __forceinline__ void store_out4(const AttendParams &p, int64_t i, float4 x, float z)
{
    if (p.out_f16 && p.out_vec) {
        *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + i) = make_uint2(pack(x.x * z, x.y * z), pack(x.z * z, x.w * z));
    } else if (p.out_vec) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + i) = make_float4(x.x * z, x.y * z, x.z * z, x.w * z);
    } else {
        store_out(p, i, x.x * z);
        store_out(p, i + 1, x.y * z);
        store_out(p, i + 2, x.z * z);
        store_out(p, i + 3, x.w * z);
    }
}

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// sum -> 1 / sum, or what an empty row gives
__device__ __forceinline__ float inverse_sum(float l, bool flash)
{
    return l == 0.0f ? (flash ? 0.0f : CUDART_NAN_F) : 1.0f / l;
}

// One query row of the warp's running softmax (a thread holds 4 of a block's 32
// keys of it; the 8 threads of a row agree on m, me and l's share is each one's own)
struct RowState {
    float m, me, l, bad;   // bad: 0, or NaN once a visible key's V block was not finite
};

// The block's 4 scores of this thread -> weights; returns the factor for the
// output so far (1 when the reference stays).
template <bool MASKED>
__device__ __forceinline__ float softmax_block(float (&s)[4], RowState &st, float ev, bool v_bad)
{
    // MASKED: natural units (a mask of the type's lowest value leaves no room for a factor); else log2
    constexpr float unit = MASKED ? kLog2e : 1.0f;
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
#pragma unroll
    for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    float orescale = 1.0f;
    if (top > -CUDART_INF_F && (st.m == -CUDART_INF_F || __fmaf_rn(top - st.m, unit, ev - st.me) > kTop)) {
        if (st.m > -CUDART_INF_F) {
            st.l *= ex2_approx((st.m - top) * unit);
            orescale = ex2_approx(__fmaf_rn(st.m - top, unit, st.me - (ev - kBias)));
        }
        st.m = top;
        st.me = ev - kBias;
    }
    if (v_bad && top > -CUDART_INF_F) st.bad = CUDART_NAN_F;
    const float m = st.m == -CUDART_INF_F ? 0.0f : st.m, up = ev - st.me;
    if constexpr (MASKED) {
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = ex2_approx(__fmaf_rn(s[i] - m, kLog2e, up));
    } else {
        // (the difference first: beside a score past 2^24 the exponent would be lost)
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = ex2_approx((s[i] - m) + up);
    }
    st.l = __fmaf_rn((s[0] + s[1]) + (s[2] + s[3]), pow2((int)-up), st.l);
    return orescale;
}

// the i-th row of a thread
template <bool DUP>
__device__ __forceinline__ int row_of(int t4, int i)
{
    const int row = (i >> 1) * 8 + 2 * t4 + (i & 1);
    return DUP ? row & 3 : row;
}

template <int D, int NG, int W, bool DUP, bool MASKED>
__global__ void __launch_bounds__(W * 32, 1) rows_kernel(const AttendParams p)
{
    using G = Rows<D, NG, W>;
    constexpr int NS = 2 * NG;   // a thread's rows: of group i / 2, 2 t4 + i % 2
    extern __shared__ __align__(128) char smem[];
    __shared__ float2 s_stat[G::W][16];
    __shared__ float s_bad[G::W][16];
    __shared__ float2 s_row[16];
    __shared__ uint2 s_q[G::q_regs ? 1 : 16][G::q_regs ? 1 : D / 4 + 4];   // (the pad: 8 rows fall on different banks)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    char *ring = smem + warp * G::ring;
    const int64_t T = (int64_t)p.n_vh * p.nb, lo = blockIdx.x * T / p.n_cta, hi = (blockIdx.x + 1) * T / p.n_cta;
    if (threadIdx.x < 2 && lo < hi) {
        // While the kernel before this one ends, HBM brings the CTA's first codes
        // to L2 (a hint: what that kernel still writes is read anew below).
        const int h = (int)(lo / p.nb), b0 = (int)(lo - (int64_t)h * p.nb);
        const int n = min(min(p.nb - b0, (int)(hi - lo)), p.l2_ahead);
        if (n > 0)
            l2_prefetch_bulk((threadIdx.x ? p.c.v : p.c.k) + ((int64_t)h * p.c.rows + (int64_t)b0 * kBlock) * D, n * kBlock * D);
    }
    bool waited = false;
    for (int64_t pos = lo; pos < hi;) {
        const int h = (int)(pos / p.nb), b0 = (int)(pos - (int64_t)h * p.nb);
        const int b1 = (int)min((int64_t)p.nb, b0 + hi - pos);
        pos += b1 - b0;
        const int nrows = p.n_new * p.r;   // (at most 4 with DUP, else 8 NG)
        const int8_t *kc = p.c.k + (int64_t)h * p.c.rows * D, *vc = p.c.v + (int64_t)h * p.c.rows * D;
        const uint32_t *ksc = reinterpret_cast<const uint32_t *>(p.c.k_scale) + (int64_t)h * (p.c.rows / kBlock);
        const uint32_t *vsc = reinterpret_cast<const uint32_t *>(p.c.v_scale) + (int64_t)h * (p.c.rows / kBlock);
        // where the queries of row g (of each group) start; the tokens of the thread's own rows
        int64_t qat[NG];
        bool have[NG];
        int tok[NS];
#pragma unroll
        for (int i = 0; i < NG; i++) {
            const int row = DUP ? g & 3 : g + 8 * i;
            have[i] = row < nrows;
            const int t = have[i] ? row / p.r : 0;
            qat[i] = t * p.q_stride + (int64_t)(h * p.r + (have[i] ? row - t * p.r : 0)) * D + t4 * 4;
        }
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int row = row_of<DUP>(t4, i);
            tok[i] = row < nrows ? row / p.r : 0;
        }
        if (!waited) {   // (nothing before it reads memory)
            pdl_wait();
            pdl_launch_dependents();
            waited = true;
        }

        // The small loads first: behind the ring's they would wait for all of them.
        // the scale words of this warp's next 32 blocks, one a lane
        uint32_t kw = 0, vw = 0;
        auto scales = [&](int b) {
            const int mine = b + lane * G::W;
            kw = mine < b1 ? ksc[mine] : 0;
            vw = mine < b1 ? vsc[mine] : 0;
        };
        scales(b0 + warp);
        // Q as the B operand: dims 4 t4 .. + 3 of each 16 (the order in which a
        // thread holds a key's codes)
        uint2 q[G::q_regs ? G::nk : 1][NG];
        if constexpr (G::q_regs) {
            if (p.q_f16 && p.q_vec) {
#pragma unroll
                for (int i = 0; i < NG; i++)
#pragma unroll
                    for (int k = 0; k < G::nk; k++)
                        q[k][i] = have[i] ? *reinterpret_cast<const uint2 *>(static_cast<const __half *>(p.q) + qat[i] + k * 16)
                                          : make_uint2(0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < NG; i++)
#pragma unroll
                    for (int k = 0; k < G::nk; k++) q[k][i] = have[i] ? load_q4(p, qat[i] + k * 16) : make_uint2(0, 0);
            }
        } else {
            for (int i = threadIdx.x; i < G::NR * (D / 4); i += G::W * 32) {
                const int row = i / (D / 4), c = i % (D / 4), t = row / p.r;
                s_q[row][c] = row < nrows ? load_q4(p, t * p.q_stride + (int64_t)(h * p.r + row - t * p.r) * D + c * 4)
                                          : make_uint2(0, 0);
            }
        }

        // this warp's blocks: b0 + warp, then every W-th; their tiles K, V, K, V ... through the ring
        int fb = b0 + warp, fs = 0;
        bool fv = false;
        auto fetch = [&] {
            if (fb < b1) {
                char *dst = ring + fs * G::tile;
                const int8_t *src = (fv ? vc : kc) + (int64_t)fb * kBlock * D;
#pragma unroll
                for (int j = 0; j < D / 16; j++) {
                    const int i = lane + 32 * j, r = i / (D / 16), c = i % (D / 16);
                    cp_async_16(dst + r * G::pitch + c * 16, src + i * 16);
                }
            }
            cp_async_commit();
            if (fv) fb += G::W;
            fv = !fv;
            if (++fs == G::E) fs = 0;
        };
        int slot = 0;
        // the next tile's address, once it has arrived; the one before it is read again by nobody
        auto next_tile = [&] {
            cp_async_wait<G::E - 2>();
            __syncwarp();
            fetch();
            const uint32_t at = smem_addr(ring + slot * G::tile);
            if (++slot == G::E) slot = 0;
            return at;
        };
#pragma unroll 1
        for (int i = 0; i < G::E - 1; i++) fetch();
        if constexpr (!G::q_regs) __syncthreads();

        RowState st[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) st[i] = RowState{-CUDART_INF_F, 0.0f, 0.0f, 0.0f};
        // dims 16 c + 2 g (of the two rows), 16 c + 2 g + 1 (of the two rows)
        float o[G::nk][NG][4];
#pragma unroll
        for (int c = 0; c < G::nk; c++)
#pragma unroll
            for (int i = 0; i < NG; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[c][i][j] = 0.0f;

        // a block's mask values, one block ahead; key j of a thread: g + 8 j
        float mk[MASKED ? NS : 1][4];
        auto masks = [&](int b) {
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int64_t key = (int64_t)b * kBlock + 8 * j + g;
                    mk[MASKED ? i : 0][j] = key < p.n_kv ? mask_value(p, tok[i], key) : -CUDART_INF_F;
                }
        };
        if (MASKED && b0 + warp < b1) masks(b0 + warp);
        for (int b = b0 + warp, n = 0; b < b1; b += G::W, n++) {
            if (n && (n & 31) == 0) scales(b);
            const uint32_t kword = __shfl_sync(0xffffffffu, kw, n & 31), vword = __shfl_sync(0xffffffffu, vw, n & 31);
            const bool k_bad = (kword & 0x7f800000u) == 0x7f800000u, v_bad = (vword & 0x7f800000u) == 0x7f800000u;
            const float ks = k_bad ? CUDART_NAN_F : pow2(scale_exp(kword)), ev = (float)scale_exp(vword);
            const int64_t key0 = (int64_t)b * kBlock;

            // S^T = K Q^T: two tiles of 16 keys, 32 dims at a time (lanes 0-7 and
            // 16-23 address keys 0-7 of a tile, the others 8-15; lanes 16-31 the
            // second 16 dims)
            const uint32_t kt = next_tile() + (lane & 15) * G::pitch + (lane >> 4) * 16;
            float acc[2][NG][4];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < NG; i++)
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[j][i][k] = 0.0f;
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                uint2 qb[2][NG];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int i = 0; i < NG; i++) {
                        if constexpr (G::q_regs) qb[k][i] = q[2 * c + k][i];
                        else qb[k][i] = s_q[g + 8 * i][(2 * c + k) * 4 + t4];
                    }
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    uint32_t w[4];
                    ldsm_x4(kt + j * 16 * G::pitch + c * 32, w[0], w[1], w[2], w[3]);
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        uint32_t x0, y0, x1, y1;
                        codes_to_half<false>(w[2 * k], x0, y0);
                        codes_to_half<false>(w[2 * k + 1], x1, y1);
#pragma unroll
                        for (int i = 0; i < NG; i++) mma_16816(acc[j][i], x0, x1, y0, y1, qb[k][i].x, qb[k][i].y);
                    }
                }
            }

            // scores, then weights
            const float cs = p.scale * ks * (MASKED ? 1.0f : kLog2e);
            float w[NS][4], orescale[NS];
            bool moved = false;
#pragma unroll
            for (int i = 0; i < NS; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float x = acc[j >> 1][i >> 1][2 * (j & 1) + (i & 1)];
                    if constexpr (MASKED) w[i][j] = mk[i][j] == -CUDART_INF_F ? mk[i][j] : __fmaf_rn(x, cs, mk[i][j]);
                    else w[i][j] = x * cs;
                }
                if (!MASKED && key0 + kBlock > p.n_past) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (key0 + 8 * j + g > p.n_past + tok[i]) w[i][j] = -CUDART_INF_F;
                }
                if (p.scores && row_of<DUP>(t4, i) < nrows && (!DUP || t4 < 2)) {
                    float *dst = p.scores + ((int64_t)h * nrows + row_of<DUP>(t4, i)) * p.nb * kBlock + key0 + g;
#pragma unroll
                    for (int j = 0; j < 4; j++) dst[8 * j] = w[i][j];
                }
                orescale[i] = softmax_block<MASKED>(w[i], st[i], ev, v_bad);
                moved |= orescale[i] != 1.0f;
            }
            if (MASKED && b + G::W < b1) masks(b + G::W);
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int c = 0; c < G::nk; c++)
#pragma unroll
                    for (int i = 0; i < NG; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) o[c][i][j] *= orescale[2 * i + (j & 1)];
            }

            // O^T += V^T W^T: two steps of 16 keys
            uint32_t pb[2][NG][2];
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int i = 0; i < NG; i++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        float e0 = w[2 * i][2 * k + x], e1 = w[2 * i + 1][2 * k + x];
                        uint32_t y = pack(e0, e1);
                        if constexpr (DUP) {
                            const __half2 hi2 = *reinterpret_cast<const __half2 *>(&y);
                            const uint32_t lo = pack(e0 - __low2float(hi2), e1 - __high2float(hi2));
                            y = t4 < 2 ? y : lo;
                        }
                        pb[k][i][x] = transpose8(y);
                    }
            const uint32_t vt = next_tile();
#pragma unroll
            for (int c = 0; c < G::nk; c++) {
                uint32_t v[4];
                ldsm_x4_t(vt + lane * G::pitch + c * 16, v[0], v[1], v[2], v[3]);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    uint32_t e0, d0, e1, d1;   // even and odd dims, keys 0-7 and 8-15 of the step
                    codes_to_half<true>(v[2 * k], e0, d0);
                    codes_to_half<true>(v[2 * k + 1], e1, d1);
#pragma unroll
                    for (int i = 0; i < NG; i++) mma_16816(o[c][i], e0, d0, e1, d1, pb[k][i][0], pb[k][i][1]);
                }
            }
        }

        // the warps' rows: (m, l) and O 2^me to shared memory, summed there
        float *os = reinterpret_cast<float *>(smem);
        cp_async_wait<0>();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NS; i++) {
            float l = st[i].l;
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
            const int row = row_of<DUP>(t4, i);
            const bool mine = !DUP || t4 < 2;
            if (g == 0 && mine) {
                s_stat[warp][row] = make_float2(st[i].m, l);
                s_bad[warp][row] = st[i].bad;
            }
            const float f = pow2((int)st[i].me);
            float *dst = os + ((int64_t)warp * G::NR + row) * D + 2 * g;
#pragma unroll
            for (int c = 0; c < G::nk; c++) {
                float x = o[c][i >> 1][i & 1], y = o[c][i >> 1][2 + (i & 1)];
                if constexpr (DUP) {   // the low halves' sums
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    y += __shfl_xor_sync(0xffffffffu, y, 2);
                }
                if (mine) *reinterpret_cast<float2 *>(dst + c * 16) = make_float2(x * f, y * f);
            }
        }
        __syncthreads();
        const bool whole = b0 == 0 && b1 == p.nb;
        const int64_t part = (int64_t)blockIdx.x + h;   // (CTA, head) pairs in order: their sum counts them
        constexpr float unit = MASKED ? kLog2e : 1.0f;
        for (int i = threadIdx.x; i < nrows * (D / 4); i += G::W * 32) {
            const int row = i / (D / 4), c = i % (D / 4) * 4;
            float M = -CUDART_INF_F;
#pragma unroll
            for (int w = 0; w < G::W; w++) M = fmaxf(M, s_stat[w][row].x);
            const float ref = M == -CUDART_INF_F ? 0.0f : M;
            float l = 0.0f;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < G::W; w++) {
                const float2 s = s_stat[w][row];
                const float f = ex2_approx((s.x - ref) * unit), bad = s_bad[w][row];
                const float4 y = *reinterpret_cast<const float4 *>(os + ((int64_t)w * G::NR + row) * D + c);
                // (a warp without a visible key: m = -inf, f = 0, its sums 0 -- or NaN, which must stay)
                l = __fmaf_rn(s.y, f, l);
                x.x = __fmaf_rn(y.x, f, x.x + bad);
                x.y = __fmaf_rn(y.y, f, x.y + bad);
                x.z = __fmaf_rn(y.z, f, x.z + bad);
                x.w = __fmaf_rn(y.w, f, x.w + bad);
            }
            if (p.cq) {
                *reinterpret_cast<float4 *>(os + G::W * G::NR * D + row * D + c) = x;
                if (c == 0) s_row[row] = make_float2(M, l);
                continue;
            }
            if (whole) store_out4(p, out_at(p, h, row, D) + c, x, inverse_sum(l, p.flash != 0));
            else *reinterpret_cast<float4 *>(p.part + (part * 16 + row) * D + c) = x;
            if (c == 0) p.stat[part * 16 + row] = make_float2(M, l);
        }
        if (p.cq) {
            // The head's CTAs are one cluster: each takes a share of the output
            // and reads the others' sums through distributed shared memory (no
            // second kernel).
            cluster_sync_all();
            for (int i = cluster_rank() * (G::W * 32) + threadIdx.x; i < nrows * (D / 4); i += p.cq * G::W * 32) {
                const int row = i / (D / 4), c = i % (D / 4) * 4;
                const uint32_t at = smem_addr(&s_row[row]), xat = smem_addr(os + G::W * G::NR * D + row * D + c);
                float2 s[kMaxCluster];
                float4 y[kMaxCluster];
                float M = -CUDART_INF_F;
#pragma unroll
                for (int k = 0; k < kMaxCluster; k++) {
                    s[k] = make_float2(-CUDART_INF_F, 0.0f);
                    y[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (k >= p.cq) continue;
                    s[k] = ld_cluster_f2(mapa(at, k));
                    y[k] = ld_cluster_f4(mapa(xat, k));
                }
#pragma unroll
                for (int k = 0; k < kMaxCluster; k++) M = fmaxf(M, s[k].x);
                const float ref = M == -CUDART_INF_F ? 0.0f : M;
                float l = 0.0f;
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < kMaxCluster; k++) {
                    const float f = ex2_approx((s[k].x - ref) * unit);
                    l = __fmaf_rn(s[k].y, f, l);
                    x.x = __fmaf_rn(y[k].x, f, x.x);
                    x.y = __fmaf_rn(y[k].y, f, x.y);
                    x.z = __fmaf_rn(y[k].z, f, x.z);
                    x.w = __fmaf_rn(y[k].w, f, x.w);
                }
                store_out4(p, out_at(p, h, row, D) + c, x, inverse_sum(l, p.flash != 0));
            }
            cluster_sync_all();   // (no CTA leaves while its sums are read)
            return;
        }
        __syncthreads();   // the next head's ring takes the shared memory
    }
}

// The CTAs of head h (the split of rows_kernel).
__device__ __forceinline__ void span_of(const AttendParams &p, int h, int &a, int &b)
{
    const int64_t T = (int64_t)p.n_vh * p.nb, x0 = (int64_t)h * p.nb, x1 = x0 + p.nb - 1;
    // CTA c holds [c T / C, (c + 1) T / C): position x is in floor(((x + 1) C - 1) / T)
    a = (int)(((x0 + 1) * p.n_cta - 1) / T);
    b = (int)(((x1 + 1) * p.n_cta - 1) / T);
}

// Joins the CTAs' partial rows: one CTA a (head, row), each of its four warps a
// quarter of the parts, kJoinU of them and their (m, l) in flight together.
// With weights, CTAs behind those add the softmax weights of 512 keys of a head.
constexpr int kJoinU = 5;

template <int D, bool MASKED>
__global__ void __launch_bounds__(128) join_kernel(const AttendParams p)
{
    constexpr float unit = MASKED ? kLog2e : 1.0f;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int R = p.n_new * p.r, n_join = p.n_vh * R;
    if ((int)blockIdx.x < n_join) {
        __shared__ float4 s_o[4][D / 4];
        __shared__ float2 s_ml[4];
        const int h = blockIdx.x / R, row = blockIdx.x - h * R;
        int a, b;
        span_of(p, h, a, b);
        const int t = row / p.r;
        const int64_t out = t * p.out_stride + (int64_t)(h * p.r + row - t * p.r) * D;
        pdl_wait();
        pdl_launch_dependents();
        if (a == b) return;   // rows_kernel wrote the output
        constexpr int V = (D / 4 + 31) / 32;
        float4 x[V];
#pragma unroll
        for (int v = 0; v < V; v++) x[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float M = -CUDART_INF_F, l = 0.0f;
        for (int c0 = a + warp; c0 <= b; c0 += 4 * kJoinU) {
            float2 s[kJoinU];
            float4 y[kJoinU][V];
#pragma unroll
            for (int u = 0; u < kJoinU; u++) {
                const int c = c0 + 4 * u;
                const int64_t at = ((int64_t)c + h) * 16 + row;
                s[u] = c <= b ? p.stat[at] : make_float2(-CUDART_INF_F, 0.0f);
#pragma unroll
                for (int v = 0; v < V; v++) {
                    y[u][v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (c <= b && lane + 32 * v < D / 4)
                        y[u][v] = *reinterpret_cast<const float4 *>(p.part + at * D + (lane + 32 * v) * 4);
                }
            }
            float top = M;
#pragma unroll
            for (int u = 0; u < kJoinU; u++) top = fmaxf(top, s[u].x);
            const float ref = top == -CUDART_INF_F ? 0.0f : top, f0 = ex2_approx((M - ref) * unit);
            M = top;
            l *= f0;
#pragma unroll
            for (int v = 0; v < V; v++) x[v] = make_float4(x[v].x * f0, x[v].y * f0, x[v].z * f0, x[v].w * f0);
#pragma unroll
            for (int u = 0; u < kJoinU; u++) {
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
#pragma unroll
        for (int v = 0; v < V; v++)
            if (lane + 32 * v < D / 4) s_o[warp][lane + 32 * v] = x[v];
        if (lane == 0) s_ml[warp] = make_float2(M, l);
        __syncthreads();
        // the four warps' sums, each relative to its own maximum
        M = fmaxf(fmaxf(s_ml[0].x, s_ml[1].x), fmaxf(s_ml[2].x, s_ml[3].x));
        const float ref = M == -CUDART_INF_F ? 0.0f : M;
        float f[4];
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            f[k] = ex2_approx((s_ml[k].x - ref) * unit);
            l = __fmaf_rn(s_ml[k].y, f[k], l);
        }
        const float z = inverse_sum(l, p.flash != 0);
        const float *o0 = reinterpret_cast<const float *>(s_o);
        for (int d = tid; d < D; d += 128) {
            float y = o0[d] * f[0];
#pragma unroll
            for (int k = 1; k < 4; k++) y = __fmaf_rn(o0[k * D + d], f[k], y);
            store_out(p, out + d, y * z);
        }
        return;
    }
    // weight[h][key] += sum over rows of e^(score - M) / Z
    __shared__ float2 s_row[16];
    const int chunks = (int)(((int64_t)p.nb * kBlock + 511) / 512);
    const int w = blockIdx.x - n_join, h = w / chunks;
    const int64_t key = (int64_t)(w - h * chunks) * 512 + tid * 4;
    int a, b;
    span_of(p, h, a, b);
    const float *src = p.scores + (int64_t)h * R * p.nb * kBlock + key;
    float *dst = p.c.weight + (int64_t)h * p.c.rows + key;
    const int64_t pitch = (int64_t)p.nb * kBlock;
    const int row = tid >> 3, sub = tid & 7;
    pdl_wait();
    pdl_launch_dependents();
    // all that is read, on its way at once: the first rows' scores, the weights so far, the parts' (m, l)
    constexpr int kAhead = 4, kParts = 3;
    float4 x[kAhead];
    float old[4];
    float2 ml[kParts];
#pragma unroll
    for (int u = 0; u < kParts; u++)
        ml[u] = row < R && a + sub + 8 * u <= b ? p.stat[((int64_t)a + sub + 8 * u + h) * 16 + row] : make_float2(-CUDART_INF_F, 0.0f);
#pragma unroll
    for (int i = 0; i < kAhead; i++)
        x[i] = key < p.n_kv && i < R ? *reinterpret_cast<const float4 *>(src + i * pitch) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 4; i++) old[i] = key + i < p.n_kv ? dst[i] : 0.0f;
    {
        float M = -CUDART_INF_F, l = 0.0f;
        auto take = [&](float M2, float l2) {
            const float top = fmaxf(M, M2);
            if (top > -CUDART_INF_F) l = __fmaf_rn(l, ex2_approx((M - top) * unit), l2 * ex2_approx((M2 - top) * unit));
            else l += l2;   // (0, or NaN)
            M = top;
        };
#pragma unroll
        for (int u = 0; u < kParts; u++) take(ml[u].x, ml[u].y);
        if (row < R)
            for (int c = a + sub + 8 * kParts; c <= b; c += 8) {
                const float2 s = p.stat[((int64_t)c + h) * 16 + row];
                take(s.x, s.y);
            }
#pragma unroll
        for (int k = 1; k < 8; k <<= 1) take(__shfl_xor_sync(0xffffffffu, M, k), __shfl_xor_sync(0xffffffffu, l, k));
        if (sub == 0) {
            const bool adds = row < R && l > 0.0f && l < CUDART_INF_F && M < CUDART_INF_F;
            s_row[row] = adds ? make_float2(M, 1.0f / l) : make_float2(0.0f, 0.0f);
        }
    }
    __syncthreads();
    if (key >= p.n_kv) return;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float2 s, float4 y) {
        if (s.y == 0.0f) return;   // (adds nothing, whatever its scores are)
        sum[0] = __fmaf_rn(ex2_approx((y.x - s.x) * unit), s.y, sum[0]);
        sum[1] = __fmaf_rn(ex2_approx((y.y - s.x) * unit), s.y, sum[1]);
        sum[2] = __fmaf_rn(ex2_approx((y.z - s.x) * unit), s.y, sum[2]);
        sum[3] = __fmaf_rn(ex2_approx((y.w - s.x) * unit), s.y, sum[3]);
    };
#pragma unroll
    for (int i = 0; i < kAhead; i++)
        if (i < R) add(s_row[i], x[i]);
#pragma unroll 4
    for (int i = kAhead; i < R; i++) add(s_row[i], *reinterpret_cast<const float4 *>(src + i * pitch));
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (key + i < p.n_kv) dst[i] = old[i] + sum[i];
}

template <int D, int NG, int W, bool DUP, bool MASKED>
cudaError_t run(const AttendParams &p, cudaStream_t st)
{
    using G = Rows<D, NG, W>;
    static Once once;
    cudaError_t e = once.on_device([] {
        return cudaFuncSetAttribute(rows_kernel<D, NG, W, DUP, MASKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::smem);
    });
    if (e == cudaSuccess) e = launch_pdl(rows_kernel<D, NG, W, DUP, MASKED>, p.n_cta, G::W * 32, G::smem, p, st, p.cq);
    if (e != cudaSuccess || p.cq) return e;
    const bool split = p.n_cta > p.n_vh || p.n_vh % p.n_cta != 0;   // else every head lies in one CTA
    if (!split && !p.scores) return cudaSuccess;
    unsigned grid = (unsigned)(p.n_vh * p.n_new * p.r);
    if (p.scores) grid += (unsigned)(p.c.H * (((int64_t)p.nb * kBlock + 511) / 512));
    return launch_pdl(join_kernel<D, MASKED>, grid, 128, 0, p, st);
}

template <int D, bool MASKED>
cudaError_t run_m(const AttendParams &p, cudaStream_t st)
{
    const int64_t rows = (int64_t)p.n_new * p.r;
    if constexpr (D < 256)
        if (rows <= 8 && p.warps == 12) return rows <= 4 ? run<D, 1, 12, true, MASKED>(p, st) : run<D, 1, 12, false, MASKED>(p, st);
    return rows <= 4 ? run<D, 1, 8, true, MASKED>(p, st) : rows <= 8 ? run<D, 1, 8, false, MASKED>(p, st) : run<D, 2, 8, false, MASKED>(p, st);
}

template <int D>
cudaError_t run_d(const AttendParams &p, cudaStream_t st)
{
    return p.mask ? run_m<D, true>(p, st) : run_m<D, false>(p, st);
}

}  // namespace

// CTAs: one an SM, about a block a warp each at least.  A CTA that crosses from
// one head to the next ends and begins a head once more, about the time of 21
// blocks: a multiple of the heads (no CTA crosses) where there are SMs for it,
// or where idling the rest costs less than that.  (32 heads: with 10 blocks for
// 21, 16k keys take 148 CTAs instead of 128, 29.9 us against 26.6; with 5 also
// 8k keys, 18.4 against 16.3.)
void rows_split(AttendParams &p)
{
    p.n_tile = 1;
    p.n_vh = p.c.H;
    p.nb = (int)((p.n_kv + kBlock - 1) / kBlock);
    constexpr int W = 8;
    const int64_t T = (int64_t)p.n_vh * p.nb;
    int64_t C = (T + W - 1) / W;
    if (C > kSMs) C = kSMs;
    // (for the same reason short heads go to CTAs of their own, in waves if need be)
    if (C < p.n_vh && (C < kSMs || p.nb <= 4 * W)) C = p.n_vh;
    if (C >= p.n_vh) {
        const int64_t up = (C + p.n_vh - 1) / p.n_vh * p.n_vh, down = C / p.n_vh * p.n_vh;
        if (up <= kSMs) C = std::min(up, T);
        else if (T / down - T / C <= 21) C = down;
    }
    // 2 to 8 CTAs a head join in their cluster instead of by a second kernel,
    // where the device holds all clusters at once (these numbers of them, by
    // the occupancy query at this shared memory): 2000 keys of 8 heads 8.0 ->
    // 5.2 us of device time.  Longer heads are not cut in 8 for it: 4000 keys
    // 7.1 us so, and 5.8 us over 128 CTAs and with the second kernel.
    constexpr int most[kMaxCluster + 1] = {0, 0, 74, 45, 33, 22, 22, 15, 15};
    p.cq = 0;
    if (!p.c.weight) {
        const int64_t q = C / p.n_vh;
        if (C % p.n_vh == 0 && q >= 2 && q <= kMaxCluster && p.n_vh <= most[q]) p.cq = (int)q;
    }
    p.n_cta = (int)C;
    // 12 warps from 28 blocks a CTA on: the loop's chain of loads, conversions
    // and products has more to hide it, the CTA's end has more rows to add.  8
    // and 12 warps: 2000 keys of 8 heads 5.2 and 5.5 us, 16k 11.2 and 11.4, 32k
    // 17.6 and 16.8, 131k 52.8 and 51.6; 16k of 32 heads of 96, 5 masked tokens,
    // 39.2 and 32.9.  (Two groups of rows, or 256 dims, do not fit 168 registers
    // a thread: 12 warps 60.9 us against 39.8, and 36.2 against 29.5.)
    p.warps = T >= 28 * C ? 12 : W;
    p.l2_ahead = W;   // a block of each warp: 20.5 -> 19.5 us at 32k keys of 8 heads; 16 gain the same, 32 nothing
}

cudaError_t launch_rows(const AttendParams &p, cudaStream_t st)
{
    switch (p.c.D) {
    case 64: return run_d<64>(p, st);
    case 96: return run_d<96>(p, st);
    case 128: return run_d<128>(p, st);
    case 256: return run_d<256>(p, st);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace q8
}  // namespace kvb
