// kv_q8_weigh.cu -- the softmax weights of a chunk's query rows, summed for each
// cached row: weight[h][k] += sum over rows of e^(t - m) / Z, with every row's
// (m, 1 / Z) known from the attention kernels.
//
// The scores are formed again as S^T = K Q^T on the tensor cores (keys on the
// 128 TMEM lanes, 128 query rows in the columns), so a thread holds one key and
// its sum never leaves its registers: no atomics, one order.  Half the products
// of the attention itself.  Without a mask 1 / Z goes into the exponent, e^(t -
// m - ln Z): one number a row to read (and one more rounding, at the size of the
// score m or of log2 Z <= 31: as the score's own, or half a step 2^-20).
// 512 tokens at 4k, 8 heads of 128: 33 us.  A pair of tiles takes 2 us, 1.1 of
// it the exponentials' units (16 a clock and SM); two warps a scheduler do not
// hide the rest of the chain (wait, read TMEM, exponentials, hand back), and the
// staging warps take 1.85 us a query tile, most of it L2's delivery.
//
// An item is (KV head, NK tiles of 128 keys); a CTA takes a range of items and
// for each walks the query tiles that see them, which L2 delivers again for
// every item: with two tiles of keys an item half as often (the same call: 37
// us with one tile, two CTAs an SM).  Each tile has its own barriers, so that one
// tile's wait falls into the other's exponentials.
//   4 warps a key tile  a key a thread: S^T from TMEM, exponentials, the sum
//   4 warps             stage: the item's codes as F16, query tiles and their
//                       rows' (m, 1 / Z)
//   1 warp              issues the MMAs, owns TMEM
#include <math_constants.h>

#include <algorithm>

#include "kv_internal.h"
#include "kv_q8_stage.cuh"

namespace kvb {
namespace q8 {
namespace {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f;

template <int D, int NK>
struct WL {
    static constexpr int threads = NK * 128 + 128 + 32;
    static constexpr int NB = (D + 63) / 64;
    static constexpr uint32_t box = 128 * 128;         // [128 rows][64 halves]
    static constexpr uint32_t tile = NB * box;         // K or Q tile
    static constexpr int n_ld = NK * D / 16;           // 16-byte loads a staging thread makes for an item's codes
    static constexpr int ctas = D == 256 || NK == 2 ? 1 : 2;   // an SM
    static constexpr int QS = NK == 2 ? 4 : 2;         // query tiles staged or in use
    static constexpr size_t o_k = 0, o_q = NK * (size_t)tile;
    static constexpr size_t o_st = o_q + QS * (size_t)tile;   // [QS][64] two rows' (-m, -m, 1 / Z, 1 / Z); without a mask four rows' -m - log2 Z
    static constexpr size_t o_off = o_st + QS * 128 * 8;      // [QS][128] where a row's queries are, -1: nowhere
    static constexpr size_t o_bar = o_off + QS * 128 * 8;
    static constexpr int n_bar = 2 + 2 * QS + 4 * NK + 1;
    static constexpr size_t o_tm = o_bar + n_bar * 8;
    static constexpr size_t bytes = o_tm + 16;
    static_assert(bytes * ctas <= 226 * 1024, "shared memory");
};

// A walk over a CTA's (item, query tile) steps, the same in every warp.
template <int NK>
struct Steps {
    int64_t item, end;
    int h, qt, n_qt;
    int64_t key0;
    int staged_h;      // the head whose only query tile is staged (-1: none)
    bool fresh;        // this step's query tile is staged anew
    __device__ __forceinline__ void begin(const AttendParams &p, int cta, int ctas)
    {
        const int64_t n = (int64_t)p.c.H * p.n_kt;
        item = cta * n / ctas;
        end = (cta + 1) * n / ctas;
        n_qt = (int)(((int64_t)p.n_new * p.r + 127) / 128);
        staged_h = -1;
        if (more()) enter(p);
    }
    __device__ __forceinline__ bool more() const { return item < end; }
    __device__ __forceinline__ void enter(const AttendParams &p)
    {
        h = (int)(item / p.n_kt);
        key0 = (item - (int64_t)h * p.n_kt) * (128 * NK);
        // tiles whose last token comes before the keys do not see them
        const int64_t tok0 = p.mask ? 0 : max((int64_t)0, key0 - p.n_past);
        qt = (int)(tok0 * p.r / 128);
        step();
    }
    __device__ __forceinline__ void step()
    {
        fresh = n_qt > 1 || staged_h != h;
        staged_h = h;
    }
    __device__ __forceinline__ bool last() const { return qt == n_qt - 1; }
    // whether the staged tile is not used after this step
    __device__ __forceinline__ bool done_with_q(const AttendParams &p) const
    {
        return n_qt > 1 || item + 1 >= end || (item + 1) / p.n_kt != h;
    }
    __device__ __forceinline__ void next(const AttendParams &p)
    {
        if (!last()) {
            qt++;
            step();
        } else {
            item++;
            if (more()) enter(p);
        }
    }
};

template <int D, int NK, bool MASKED>
__global__ void __launch_bounds__(WL<D, NK>::threads, WL<D, NK>::ctas) weigh_kernel(const AttendParams p)
{
    using L = WL<D, NK>;
    constexpr int QS = L::QS, kStage = NK * 4, kIssue = kStage + 4;   // the first staging warp, the issuing warp
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + L::o_bar);
    uint64_t *k_full = bar, *k_empty = bar + 1, *q_full = bar + 2, *q_empty = q_full + QS, *s_full = q_empty + QS;
    uint64_t *s_empty = s_full + 2 * NK, *drain = s_empty + 2 * NK;   // [buffer][key tile]
    uint32_t *tm_slot = reinterpret_cast<uint32_t *>(smem + L::o_tm);
    volatile int *flag = reinterpret_cast<volatile int *>(smem + L::o_tm + 8);
    float4 *row_st = reinterpret_cast<float4 *>(smem + L::o_st);
    int64_t *row_off = reinterpret_cast<int64_t *>(smem + L::o_off);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(k_full, p.inject == 2 ? 5 : 4);   // (test hook: one arrival too many is waited for)
        mbar_init(k_empty, 1);
        for (int i = 0; i < QS; i++) {
            mbar_init(&q_full[i], 4);
            mbar_init(&q_empty[i], 1 + kStage);   // the MMAs that read it, and the warps that read its rows' numbers
        }
        for (int i = 0; i < 2 * NK; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], 4);
        }
        mbar_init(drain, 1);
        *flag = 0;
        fence_mbar_init();
    }
    if (warp == kIssue) {
        tmem_alloc(tm_slot, 256 * NK);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tm_slot;
    Steps<NK> w;
    w.begin(p, blockIdx.x, gridDim.x);
    pdl_wait();
    pdl_launch_dependents();
    auto wait = [&](uint64_t *b, uint32_t par) {
        if (mbar_wait_ab(b, par, p.limit_ns, flag)) return true;
        give_up(p.error, flag, 8u);
        return false;
    };

    bool ok = true;
    int q = -1, s = 0, items = 0;   // query tiles staged (the present one's number), steps, items begun
    if (warp < kStage) {
        const int kt = warp >> 2;   // key tile of the item
        const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + kt * 128;
        float sum = 0.0f, c = 0.0f;
        int first = 0;   // the first row that sees the thread's key (without a mask)
        int64_t now = -1;
        // where a wait of the chunk's kernel expired, rows' (m, 1 / Z) are not this call's: nothing is added then
        unsigned lost = 0;
        for (int i = lane; i < p.n_cta; i += 32) lost |= p.gave_up[i];
        const bool keeps = !__any_sync(0xffffffffu, lost);
        for (; ok && w.more(); s++) {
            if (w.fresh) q++;
            const int64_t key = w.key0 + tid;   // (the warps of a tile are in lane order)
            const int qs = q % QS;
            if (w.item != now) {
                // (key 0 of the item is a row of the cache: the block of a lane past the cache is the last one)
                now = w.item;
                const int64_t blk = min(key / kBlock, p.c.rows / kBlock - 1);
                const uint32_t kw = reinterpret_cast<const uint32_t *>(p.c.k_scale)[(int64_t)w.h * (p.c.rows / kBlock) + blk];
                c = p.scale * pow2(scale_exp(kw)) * (MASKED ? 1.0f : kLog2e);
                first = (int)max((int64_t)0, min((int64_t)p.n_new, key - p.n_past)) * p.r;
            }
            ok = __all_sync(0xffffffffu, wait(&q_full[qs], (q / QS) & 1) && wait(&s_full[(s & 1) * NK + kt], (s >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const float4 *st = row_st + qs * 64;
            const int row0 = w.qt * 128, n_rows = min(128, p.n_new * p.r - row0);
            const bool in = key < p.n_kv;
            uint64_t part = 0ull;   // two sums
            const uint64_t c2 = pk2(c, c);
            // N rows' scores, and with a mask its values
            constexpr int N = MASKED ? 16 : 32;
            float mk[MASKED ? N : 1];
            auto rows = [&](int ch, uint32_t (&v)[N]) {
                if constexpr (MASKED) {
                    float a = 0.0f;
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const float4 y4 = st[(ch * N + e) / 2];
                        const float m = e & 1 ? y4.y : y4.x, y = e & 1 ? y4.w : y4.z;
                        const float x = ex2_approx((__fmaf_rn(__uint_as_float(v[e]), c, mk[e]) + m) * kLog2e);
                        a = y == 0.0f ? a : __fmaf_rn(x, y, a);   // (1 / Z = 0: its mask may be infinite)
                    }
                    part = add2(part, pk2(a, 0.0f));
                } else {
                    const int hide = first - row0 - ch * N;   // rows of these that do not see the key
                    if (__all_sync(0xffffffffu, hide >= N)) return;
                    if (__any_sync(0xffffffffu, hide > 0)) {
#pragma unroll
                        for (int e = 0; e < N; e++)
                            if (e < hide) v[e] = __float_as_uint(-CUDART_INF_F);
                    }
                    uint64_t s0 = 0ull, s1 = 0ull;
#pragma unroll
                    for (int e = 0; e < N / 4; e++) {
                        const float4 y = st[ch * (N / 4) + e];
                        const float2 a = up2(fma2(pk2(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1])), c2, pk2(y.x, y.y)));
                        const float2 b = up2(fma2(pk2(__uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3])), c2, pk2(y.z, y.w)));
                        s0 = add2(s0, pk2(ex2_approx(a.x), ex2_approx(a.y)));
                        s1 = add2(s1, pk2(ex2_approx(b.x), ex2_approx(b.y)));
                    }
                    part = add2(part, add2(s0, s1));
                }
            };
            const uint32_t at = tS + (s & 1) * (128 * NK);
            if constexpr (MASKED) {
                int tok = row0 / p.r, j = row0 - tok * p.r;   // of the next row
                const void *src = p.mask;
#pragma unroll 1
                for (int ch = 0; ch * N < n_rows; ch++) {
                    uint32_t v[N], raw[N];
                    tmem_ld16(at + ch * N, v);
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        // (at clamped places, so that the loads are in flight together; a token's rows read the same values, from L1)
                        const int64_t i = min(tok, p.n_new - 1) * p.mask_stride + min(key, p.n_kv - 1);
                        raw[e] = p.mask_f16 ? static_cast<const unsigned short *>(src)[i] : static_cast<const uint32_t *>(src)[i];
                        if (++j == p.r) {
                            j = 0;
                            tok++;
                        }
                    }
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < N; e++)
                        mk[e] = !in ? -CUDART_INF_F : p.mask_f16 ? __half2float(__ushort_as_half((unsigned short)raw[e])) : __uint_as_float(raw[e]);
                    rows(ch, v);
                }
            } else if constexpr (L::ctas == 2) {   // (two CTAs an SM: 96 registers a thread)
#pragma unroll 1
                for (int ch = 0; ch * N < n_rows; ch++) {
                    uint32_t v[N];
                    tmem_ld32(at + ch * N, v);
                    tmem_wait_ld();
                    rows(ch, v);
                }
            } else {
                // the next rows' scores on their way during the exponentials
                uint32_t v[2][N];
                tmem_ld32(at, v[0]);
#pragma unroll
                for (int ch = 0; ch < 128 / N; ch++) {
                    if (ch * N >= n_rows) break;
                    tmem_wait_ld();
                    if (ch * N + N < n_rows) tmem_ld32(at + ch * N + N, v[(ch + 1) & 1]);
                    rows(ch, v[ch & 1]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&s_empty[(s & 1) * NK + kt]);
                if (w.done_with_q(p)) mbar_arrive(&q_empty[qs]);
            }
            {
                const float2 x = up2(part);
                sum += x.x + x.y;
            }
            if (w.last()) {
                if (in && keeps) p.c.weight[(int64_t)w.h * p.c.rows + key] += sum;
                sum = 0.0f;
            }
            w.next(p);
        }
    } else if (warp < kIssue) {
        const int t = tid - kStage * 32;
        uint4 buf[L::n_ld];
        auto load = [&](int64_t item) {
            const int h = (int)(item / p.n_kt);
            const int64_t key0 = (item - (int64_t)h * p.n_kt) * (128 * NK);
            const uint4 *src = reinterpret_cast<const uint4 *>(p.c.k + ((int64_t)h * p.c.rows + key0) * D);
#pragma unroll
            for (int j = 0; j < L::n_ld; j++) {
                const int i = t + 128 * j;
                buf[j] = key0 + i / (D / 16) < p.c.rows ? src[i] : make_uint4(0, 0, 0, 0);
            }
        };
        if (w.more()) load(w.item);
        auto all_wait = [&](uint64_t *b, uint32_t par) { return __all_sync(0xffffffffu, wait(b, par)); };
        const uint32_t sk = smem_addr(smem + L::o_k), sq = smem_addr(smem + L::o_q);
        bool ahead = false;   // `next` holds the numbers of this thread's row of the next tile
        float2 next = make_float2(0.0f, 0.0f);
        ok = !(p.inject == 3 && warp == kStage);   // (test hook: this warp alone gives up)
        // (a warp that gave up comes to the barrier below like the others, and all four leave together)
        for (int64_t now = -1; w.more(); w.next(p)) {
            if (ok && w.item != now && items > 0) ok = all_wait(k_empty, (items - 1) & 1);
            if (ok && w.item != now) {
#pragma unroll
                for (int j = 0; j < L::n_ld; j++) {
                    const int i = t + 128 * j;
                    const int r = i / (D / 16);
                    store_codes(sk + (r >> 7) * L::tile, L::box, r & 127, i % (D / 16), buf[j]);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full);
                now = w.item;
                items++;
                if (w.item + 1 < w.end) load(w.item + 1);
            }
            if (!w.fresh) continue;
            q++;
            const int qs = q % QS;
            if (ok && q >= QS) ok = all_wait(&q_empty[qs], (q / QS - 1) & 1);
            const int row0 = w.qt * 128, R = p.n_new * p.r;
            const float2 *stat = p.row_stat + (int64_t)w.h * R + row0;
            int64_t *off = row_off + qs * 128;
            if (ok) {
                // a row that adds nothing has 1 / Z = 0: its queries are zeros, so that its products are finite
                const float2 y = ahead ? next : row0 + t < R ? stat[t] : make_float2(0.0f, 0.0f);
                const int tok = (row0 + t) / p.r, j = row0 + t - tok * p.r;
                if constexpr (MASKED) {
                    float *rs = reinterpret_cast<float *>(row_st + qs * 64 + t / 2) + (t & 1);
                    rs[0] = -y.x;
                    rs[2] = y.y;
                } else {
                    reinterpret_cast<float *>(row_st + qs * 64)[t] = log2f(y.y) - y.x;   // (1 / Z = 0: -inf)
                }
                off[t] = y.y != 0.0f ? tok * p.q_stride + (int64_t)(w.h * p.r + j) * D : -1;
            }
            if (named_sync_or(1, 128, !ok)) break;
            stage_queries<D>(p, sq + qs * L::tile, L::box, off, t);
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[qs]);
            // (not before the fence, which waits for loads in flight)
            ahead = !w.last();
            if (ahead) next = row0 + 128 + t < R ? stat[128 + t] : make_float2(0.0f, 0.0f);
        }
    } else if (lane == 0) {
        constexpr uint32_t id = idesc_f16_f32(128, 128, false);
        const uint32_t sk = smem_addr(smem + L::o_k), sq = smem_addr(smem + L::o_q);
        for (int64_t now = -1; ok && w.more(); s++, w.next(p)) {
            if (w.item != now) {
                if (!(ok = wait(k_full, items & 1))) break;
                now = w.item;
                items++;
            }
            if (w.fresh) {
                q++;
                if (!(ok = wait(&q_full[q % QS], (q / QS) & 1))) break;
            }
#pragma unroll
            for (int k = 0; k < NK; k++) {
                const int buf = (s & 1) * NK + k;
                if (s >= 2 && !(ok = wait(&s_empty[buf], ((s >> 1) - 1) & 1))) break;
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                    const uint32_t off = (kk >> 2) * L::box + (kk & 3) * 32;
                    umma_ss(tmem + buf * 128, sdesc_k_sw128(sk + k * L::tile + off), sdesc_k_sw128(sq + (q % QS) * L::tile + off), id,
                            kk > 0);
                }
                umma_commit(&s_full[buf]);
            }
            if (!ok) break;
            if (w.done_with_q(p)) umma_commit(&q_empty[q % QS]);
            if (w.last()) umma_commit(k_empty);
        }
        umma_commit(drain);
        mbar_wait(drain, 0, p.limit_ns);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssue) {
        tc_fence_after();
        tmem_dealloc(tmem, 256 * NK);
    }
}

template <int D, int NK, bool MASKED>
cudaError_t run(AttendParams p, cudaStream_t st)
{
    using L = WL<D, NK>;
    static Once once;
    cudaError_t e = once.on_device([] {
        return cudaFuncSetAttribute(weigh_kernel<D, NK, MASKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::bytes);
    });
    if (e != cudaSuccess) return e;
    p.n_kt = (int)((p.n_kv + 128 * NK - 1) / (128 * NK));
    const unsigned grid = (unsigned)std::min<int64_t>((int64_t)p.c.H * p.n_kt, kSMs * L::ctas);
    return launch_pdl(weigh_kernel<D, NK, MASKED>, grid, L::threads, L::bytes, p, st);
}

template <int D, bool MASKED>
cudaError_t run_d(const AttendParams &p, cudaStream_t st)
{
    // two tiles of keys an item where that leaves most SMs one (at head_dim 256 their codes would not fit)
    if constexpr (D < 256)
        if (p.c.H * ((p.n_kv + 255) / 256) >= kSMs / 2) return run<D, 2, MASKED>(p, st);
    return run<D, 1, MASKED>(p, st);
}

}  // namespace

cudaError_t launch_weigh(const AttendParams &p, cudaStream_t st)
{
    switch (p.c.D) {
    case 64: return p.mask ? run_d<64, true>(p, st) : run_d<64, false>(p, st);
    case 96: return p.mask ? run_d<96, true>(p, st) : run_d<96, false>(p, st);
    case 128: return p.mask ? run_d<128, true>(p, st) : run_d<128, false>(p, st);
    case 256: return p.mask ? run_d<256, true>(p, st) : run_d<256, false>(p, st);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace q8
}  // namespace kvb
