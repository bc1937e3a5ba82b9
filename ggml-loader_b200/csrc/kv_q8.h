// kv_q8.h -- the 8-bit cache: what its kernels and the C entry points share.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace kvb {
namespace q8 {

constexpr int kBlock = 32;   // rows that share a scale (KV_Q8_BLOCK)
constexpr int kSMs = 148;    // the most CTAs a split uses
constexpr uint64_t kLimitNs = 1000000000ull;   // AttendParams::limit_ns of a call on the caller's buffers: 1 s
constexpr int kExpMin = -24, kExpMax = 9;   // a scale is 2^e with e in this range

struct Cache {
    int8_t *k, *v;              // [H][rows][D]
    float *k_scale, *v_scale;   // [H][rows / kBlock]
    float *weight;              // [H][rows] or null
    int64_t rows;
    int32_t H, D;
};

struct StoreParams {
    Cache c;
    const void *k, *v;
    int64_t k_stride, v_stride;   // elements a token
    int64_t row0;
    int32_t n_new;
    int32_t f16;   // 1: __half rows, 0: float rows
    int32_t vec;   // every row starts on a 16-byte boundary
};
cudaError_t launch_store(const StoreParams &p, cudaStream_t st);

struct LoadParams {
    Cache c;
    void *k, *v;   // either may be null
    int64_t stride;
    int64_t row0, n;
    int32_t f16, vec;
};
cudaError_t launch_load(const LoadParams &p, cudaStream_t st);

struct EvictParams {
    Cache src, dst;
    int64_t n_rows, keep, recent;
    int32_t *kept;   // [H][keep]
};
cudaError_t launch_evict(const EvictParams &p, cudaStream_t st);

struct AttendParams {
    Cache c;
    int32_t Hq, r;          // query heads, query heads a KV head
    int64_t n_past, n_kv;   // n_kv = n_past + n_new
    int32_t n_new;
    const void *q;
    int64_t q_stride;
    int32_t q_f16, q_vec;   // q_vec: every head starts on a 16-byte boundary
    const void *mask;       // null: causal
    int64_t mask_stride;
    int32_t mask_f16;
    int32_t flash;          // a row without a visible key gives 0 (else NaN)
    void *out;
    int64_t out_stride;
    int32_t out_f16, out_vec;
    float scale;
    // scratch of the workspace, set by launch_attend
    int32_t nb;             // blocks of kBlock keys: ceil(n_kv / kBlock)
    int32_t n_tile;         // chunk: query-row tiles a CTA holds (rows: 1)
    int32_t n_vh;           // what CTAs work on at a time: KV heads, or (chunk) pairs of one and a block, H * n_blk
    int32_t n_cta;
    int32_t cq;             // rows: CTAs of a head's cluster, 0: no clusters
    int32_t warps;          // rows: a CTA's, 8 or 12
    int32_t l2_ahead;       // rows: blocks a CTA asks for in L2 while the kernel before ends
    int32_t tok_tile, tok_blk, n_blk;   // chunk: tokens of a query tile and of a CTA's tiles, such blocks
    int64_t subs;           // chunk: sub-tiles of 64 keys of one KV head, over its blocks
    int32_t gap;            // chunk: what a pair's beginning counts for where the work is cut, in sub-tiles
    float *part;            // [n_cta + n_vh][rows][D] partial outputs of a (CTA, head or pair); rows: 16,
                            // or a chunk block's 128 * n_tile
    float2 *stat;           // [n_cta + n_vh][rows] their (maximum, sum)
    float *scores;          // [H][n_new * r][nb * kBlock] or null
    float2 *row_stat;       // [H][n_new * r] (maximum, 1 / sum or 0) or null
    unsigned *gave_up;      // [n_cta] whether a wait of the chunk's CTA expired, or null (no weights)
    int32_t n_kt;           // weigh: a KV head's items of 128 or 256 keys
    unsigned *error;        // the record of waits that expired: a context's, or null for the device's
    uint64_t limit_ns;      // bound of every wait in the chunk's and the weights' kernels
    int32_t inject;         // test hook (kv_debug_inject): which wait's partner stays away
};
// bytes of workspace (a function of the sizes alone)
uint64_t attend_workspace(const AttendParams &p);
cudaError_t launch_attend(AttendParams p, void *ws, cudaStream_t st);

// kv_q8_rows.cu: the split of a call over CTAs, and its kernels
void rows_split(AttendParams &p);
cudaError_t launch_rows(const AttendParams &p, cudaStream_t st);
// kv_q8_chunk.cu: the same for more than 16 query rows a KV head
void chunk_split(AttendParams &p);
cudaError_t launch_chunk(const AttendParams &p, cudaStream_t st);
// kv_q8_weigh.cu: a chunk's softmax weights into the cache's accumulator
cudaError_t launch_weigh(const AttendParams &p, cudaStream_t st);
// the current device's record of waits that expired, of calls on the callers' buffers: its address
cudaError_t error_word(unsigned **dev);
// a record's bits since the last call, behind what `st` holds (record: two words, one of them for the answer's way back)
cudaError_t take_error(unsigned *record, cudaStream_t st, unsigned *word);

// kernels that the calling thread has launched (launch_pdl counts them)
int64_t &launched();

// Runs a function once a device (a kernel's attributes last); devices past 63 run it every time.
struct Once {
    std::atomic<uint64_t> done{0};
    template <class F>
    cudaError_t on_device(F &&f)
    {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
        e = f();
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
        return e;
    }
};

}  // namespace q8
}  // namespace kvb
