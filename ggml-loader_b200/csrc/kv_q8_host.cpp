// kv_q8_host.cpp -- the C entry points of the 8-bit cache (include/kv_api.h):
// argument checks and launches.  They allocate nothing and keep no state but
// the device's record of waits that expired.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "kv_api.h"
#include "kv_internal.h"
#include "kv_q8.h"

namespace {

using kvb::q8::Cache;

int fail(int code, const char *fmt, ...)
{
    char msg[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    return kvb::set_last_error(code, msg);
}

int cuda_rc(cudaError_t e, const char *what)
{
    return e == cudaSuccess ? KV_OK : fail(KV_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_cache(const char *what, const kv_q8_cache *c, Cache &out)
{
    if (!c) return fail(KV_E_ARG, "%s: cache is NULL", what);
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256)
        return fail(KV_E_ARG, "%s: head_dim %d unsupported (64, 96, 128, 256)", what, c->head_dim);
    if (c->n_head_kv <= 0 || c->n_head_kv > 1024) return fail(KV_E_ARG, "%s: n_head_kv outside [1, 1024]", what);
    if (c->rows <= 0 || c->rows % KV_Q8_BLOCK != 0 || c->rows > ((int64_t)1 << 31) - KV_Q8_BLOCK)
        return fail(KV_E_ARG, "%s: rows must be a positive multiple of %d below 2^31", what, KV_Q8_BLOCK);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(KV_E_ARG, "%s: a cache buffer is NULL", what);
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return fail(KV_E_ARG, "%s: codes must be 16-byte aligned", what);
    if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->weight, 4))
        return fail(KV_E_ARG, "%s: scales and weights must be 4-byte aligned", what);
    out = Cache{c->k, c->v, c->k_scale, c->v_scale, c->weight, c->rows, c->n_head_kv, c->head_dim};
    return KV_OK;
}

int check_type(const char *what, int32_t type)
{
    return type == KV_F32 || type == KV_F16 ? KV_OK : fail(KV_E_ARG, "%s: unknown element type %d", what, type);
}

// an element pointer and a row stride of that type: aligned for its elements;
// vec: every row (and head) starts on a 16-byte boundary
bool elem_aligned(const void *p, int32_t type) { return aligned(p, type == KV_F16 ? 2 : 4); }
bool vec_ok(const void *p, int64_t stride, int32_t type)
{
    return aligned(p, 16) && stride % (type == KV_F16 ? 8 : 4) == 0;
}

int check_rows(const char *what, const Cache &c, int64_t row0, int64_t n)
{
    if (row0 < 0 || n <= 0 || row0 > c.rows || n > c.rows - row0)
        return fail(KV_E_RANGE, "%s: rows [%lld, +%lld) outside the cache's %lld", what, (long long)row0, (long long)n,
                    (long long)c.rows);
    return KV_OK;
}

// the sizes of an attend call (shared with the workspace query)
int attend_sizes(const kv_q8_cache *cache, int32_t n_head, int64_t n_past, int32_t n_new, kvb::q8::AttendParams &p)
{
    const char *what = "kv_q8_attend";
    int rc = check_cache(what, cache, p.c);
    if (rc) return rc;
    if (n_head <= 0 || n_head % p.c.H != 0 || n_head / p.c.H > 128)
        return fail(KV_E_ARG, "%s: n_head must be a multiple of n_head_kv, at most 128 times it", what);
    if (n_new <= 0 || n_new > 65535) return fail(KV_E_RANGE, "%s: n_new outside [1, 65535]", what);
    rc = check_rows(what, p.c, n_past, n_new);
    if (rc) return rc;
    p.Hq = n_head;
    p.r = n_head / p.c.H;
    p.n_past = n_past;
    p.n_new = n_new;
    p.n_kv = n_past + n_new;
    return KV_OK;
}

}  // namespace

int kv_q8_store(const kv_q8_cache *cache, int64_t row0, int32_t n_new, const void *k, int64_t k_stride,
                const void *v, int64_t v_stride, int32_t type, void *stream)
{
    const char *what = "kv_q8_store";
    kvb::q8::StoreParams p{};
    int rc = check_cache(what, cache, p.c);
    if (rc == KV_OK) rc = check_type(what, type);
    if (rc == KV_OK) rc = check_rows(what, p.c, row0, n_new);
    if (rc) return rc;
    if (!k || !v) return fail(KV_E_ARG, "%s: k and v are required", what);
    if (!elem_aligned(k, type) || !elem_aligned(v, type)) return fail(KV_E_ARG, "%s: misaligned k or v", what);
    const int64_t wide = (int64_t)p.c.H * p.c.D;
    if (n_new > 1 && (k_stride < wide || v_stride < wide))
        return fail(KV_E_ARG, "%s: row strides shorter than a token's heads", what);
    p.k = k;
    p.v = v;
    p.k_stride = n_new > 1 ? k_stride : 0;   // (one row: no stride is used)
    p.v_stride = n_new > 1 ? v_stride : 0;
    p.row0 = row0;
    p.n_new = n_new;
    p.f16 = type == KV_F16;
    p.vec = vec_ok(k, p.k_stride, type) && vec_ok(v, p.v_stride, type);
    return cuda_rc(kvb::q8::launch_store(p, static_cast<cudaStream_t>(stream)), what);
}

int kv_q8_load(const kv_q8_cache *cache, int64_t row0, int64_t n, void *k_out, void *v_out, int64_t stride,
               int32_t type, void *stream)
{
    const char *what = "kv_q8_load";
    kvb::q8::LoadParams p{};
    int rc = check_cache(what, cache, p.c);
    if (rc == KV_OK) rc = check_type(what, type);
    if (rc == KV_OK) rc = check_rows(what, p.c, row0, n);
    if (rc) return rc;
    if (!k_out && !v_out) return fail(KV_E_ARG, "%s: no output", what);
    if (!elem_aligned(k_out, type) || !elem_aligned(v_out, type)) return fail(KV_E_ARG, "%s: misaligned output", what);
    if (n > 1 && stride < (int64_t)p.c.H * p.c.D)
        return fail(KV_E_ARG, "%s: stride shorter than a token's heads", what);
    p.k = k_out;
    p.v = v_out;
    p.stride = n > 1 ? stride : 0;
    p.row0 = row0;
    p.n = n;
    p.f16 = type == KV_F16;
    p.vec = vec_ok(k_out, p.stride, type) && vec_ok(v_out, p.stride, type);
    return cuda_rc(kvb::q8::launch_load(p, static_cast<cudaStream_t>(stream)), what);
}

uint64_t kv_q8_attend_workspace(const kv_q8_cache *cache, int32_t n_head, int64_t n_past, int32_t n_new)
{
    kvb::q8::AttendParams p{};
    return attend_sizes(cache, n_head, n_past, n_new, p) == KV_OK ? kvb::q8::attend_workspace(p) : 0;
}

int kv_q8_attend(const kv_q8_cache *cache, int32_t n_head, int64_t n_past, int32_t n_new,
                 const void *q, int64_t q_stride, int32_t q_type,
                 const void *mask, int32_t mask_type, int64_t mask_stride, uint32_t flags,
                 void *out, int64_t out_stride, int32_t out_type,
                 void *workspace, uint64_t workspace_bytes, void *stream)
{
    const char *what = "kv_q8_attend";
    kvb::q8::AttendParams p{};
    int rc = attend_sizes(cache, n_head, n_past, n_new, p);
    if (rc == KV_OK) rc = check_type(what, q_type);
    if (rc == KV_OK) rc = check_type(what, out_type);
    if (rc) return rc;
    if (!q || !out || !workspace) return fail(KV_E_ARG, "%s: q, out and workspace are required", what);
    if (!elem_aligned(q, q_type) || !elem_aligned(out, out_type))
        return fail(KV_E_ARG, "%s: misaligned q or out", what);
    if (!aligned(workspace, 256)) return fail(KV_E_ARG, "%s: workspace must be 256-byte aligned", what);
    const int64_t wide = (int64_t)n_head * p.c.D;
    if (n_new > 1 && (q_stride < wide || out_stride < wide))
        return fail(KV_E_ARG, "%s: row strides shorter than a token's heads", what);
    if (mask) {
        if (mask_type != KV_MASK_F32 && mask_type != KV_MASK_F16)
            return fail(KV_E_ARG, "%s: unknown mask type %d", what, mask_type);
        if (n_new > 1 && mask_stride < p.n_kv)
            return fail(KV_E_ARG, "%s: mask_stride %lld < the %lld keys attended", what, (long long)mask_stride,
                        (long long)p.n_kv);
        if (!aligned(mask, mask_type == KV_MASK_F16 ? 2 : 4)) return fail(KV_E_ARG, "%s: misaligned mask", what);
    }
    if ((flags & ~(uint32_t)KV_ATTN_FLASH) != 0) return fail(KV_E_ARG, "%s: unknown flags 0x%x", what, flags);
    const uint64_t need = kvb::q8::attend_workspace(p);
    if (workspace_bytes < need)
        return fail(KV_E_RANGE, "%s: workspace of %llu bytes, %llu needed", what, (unsigned long long)workspace_bytes,
                    (unsigned long long)need);
    p.q = q;
    p.q_stride = n_new > 1 ? q_stride : 0;
    p.q_f16 = q_type == KV_F16;
    p.q_vec = vec_ok(q, p.q_stride, q_type);
    p.mask = mask;
    p.mask_stride = n_new > 1 ? mask_stride : 0;
    p.mask_f16 = mask_type == KV_MASK_F16;
    p.flash = (flags & KV_ATTN_FLASH) != 0;
    p.out = out;
    p.out_stride = n_new > 1 ? out_stride : 0;
    p.out_f16 = out_type == KV_F16;
    p.out_vec = vec_ok(out, p.out_stride, out_type);
    p.scale = 1.0f / sqrtf((float)p.c.D);
    p.limit_ns = kvb::q8::kLimitNs;
    return cuda_rc(kvb::q8::launch_attend(p, workspace, static_cast<cudaStream_t>(stream)), what);
}

int kv_q8_status(void *stream)
{
    const char *what = "kv_q8_status";
    int rc = cuda_rc(cudaStreamSynchronize(static_cast<cudaStream_t>(stream)), what);
    unsigned word = 0, *record = nullptr;
    if (rc == KV_OK) rc = cuda_rc(kvb::q8::error_word(&record), what);
    if (rc == KV_OK) {
        static std::mutex one;   // (one word a device for the answer's way back)
        std::lock_guard<std::mutex> lock(one);
        rc = cuda_rc(kvb::q8::take_error(record, static_cast<cudaStream_t>(stream), &word), what);
    }
    if (rc == KV_OK && word)
        return fail(KV_E_TIMEOUT, "%s: a wait in an attention kernel expired (bits 0x%x); its outputs are not valid", what,
                    word);
    return rc;
}

int kv_q8_evict(const kv_q8_cache *src, int64_t n_rows, int64_t keep, int64_t recent,
                const kv_q8_cache *dst, int32_t *kept, void *stream)
{
    const char *what = "kv_q8_evict";
    kvb::q8::EvictParams p{};
    int rc = check_cache(what, src, p.src);
    if (rc == KV_OK) rc = check_cache(what, dst, p.dst);
    if (rc) return rc;
    if (p.src.H != p.dst.H || p.src.D != p.dst.D)
        return fail(KV_E_ARG, "%s: src and dst differ in n_head_kv or head_dim", what);
    if (!p.src.weight) return fail(KV_E_ARG, "%s: src keeps no weights", what);
    if (!kept || !aligned(kept, 4)) return fail(KV_E_ARG, "%s: kept is required, 4-byte aligned", what);
    if (keep < 1 || recent < 0 || recent > keep || keep > n_rows)
        return fail(KV_E_ARG, "%s: 0 <= recent <= keep <= n_rows and keep >= 1 are required", what);
    if (n_rows > p.src.rows || keep > p.dst.rows) return fail(KV_E_RANGE, "%s: more rows than a cache holds", what);
    // the buffers of src and dst (and kept) must not overlap
    struct Span { const void *p; uint64_t n; };
    auto spans = [](const Cache &c, Span (&s)[5]) {
        const uint64_t codes = (uint64_t)c.H * c.rows * c.D, scales = (uint64_t)c.H * (c.rows / KV_Q8_BLOCK) * 4;
        s[0] = {c.k, codes};
        s[1] = {c.v, codes};
        s[2] = {c.k_scale, scales};
        s[3] = {c.v_scale, scales};
        s[4] = {c.weight, c.weight ? (uint64_t)c.H * c.rows * 4 : 0};
    };
    Span a[5], b[6];
    spans(p.src, a);
    {
        Span d[5];
        spans(p.dst, d);
        for (int i = 0; i < 5; i++) b[i] = d[i];
        b[5] = {kept, (uint64_t)p.src.H * keep * 4};
    }
    for (const Span &x : a)
        for (const Span &y : b) {
            const uintptr_t x0 = reinterpret_cast<uintptr_t>(x.p), y0 = reinterpret_cast<uintptr_t>(y.p);
            if (x.n && y.n && x0 < y0 + y.n && y0 < x0 + x.n)
                return fail(KV_E_ARG, "%s: a buffer of dst (or kept) overlaps one of src", what);
        }
    p.n_rows = n_rows;
    p.keep = keep;
    p.recent = recent;
    p.kept = kept;
    return cuda_rc(kvb::q8::launch_evict(p, static_cast<cudaStream_t>(stream)), what);
}
