// kv_q8_attend.cpp -- attention over the 8-bit cache: which kernels a call
// takes, and its workspace.
#include <algorithm>

#include "kv_q8.h"

namespace kvb {
namespace q8 {
namespace {

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
    p.gave_up = nullptr;
    if (p.c.weight && !chunk) p.scores = reinterpret_cast<float *>(take(p.c.H * rows * p.nb * kBlock * sizeof(float)));
    if (p.c.weight && chunk) {
        p.row_stat = reinterpret_cast<float2 *>(take(p.c.H * rows * sizeof(float2)));
        p.gave_up = reinterpret_cast<unsigned *>(take(kSMs * sizeof(unsigned)));
    }
    return n;
}

}  // namespace

int64_t &launched()
{
    static thread_local int64_t n = 0;
    return n;
}

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
    if ((int64_t)p.n_new * p.r <= 16) return launch_rows(p, st);
    cudaError_t e = p.error ? cudaSuccess : error_word(&p.error);
    if (e == cudaSuccess) e = launch_chunk(p, st);
    return e != cudaSuccess || !p.row_stat ? e : launch_weigh(p, st);
}

}  // namespace q8
}  // namespace kvb
