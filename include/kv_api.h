/*
 * kv_api.h -- C ABI of the B200 KV-cache append + attention path.
 *
 * This is the drop-in boundary for GGML-Loader's per-layer KV-cache hot path
 * (src/model.cpp in the reference).  A caller that today builds the ggml op
 * sequence in build_graph() for the phi3 / qwen2 / qwen3 / llama architectures
 * calls, per layer:
 *
 *     kv_append(ctx, layer, n_past, n_new, q, k, v, ...)   -- replaces the
 *         QK-Norm (model.cpp:1382-1387), ggml_rope_ext (1389-1404) and the
 *         ggml_cpy of K/V into the cache view (1406-1414);
 *     kv_attend(ctx, layer, n_past, n_new, out, ...)        -- replaces the
 *         attention over cache rows [0, n_past+n_new): ggml_mul_mat(K,Q),
 *         ggml_soft_max_ext with the causal mask, ggml_mul_mat(V^T, KQ) and the
 *         output permute (1416-1445), or the flash-attn branch (1426-1434).
 *
 * and at start-up kv_alloc() in place of init_kv_cache() (model.cpp:821-867),
 * with the context auto-sizing of auto_n_ctx() (model.cpp:1002-1059) computed
 * from free HBM instead of /proc/meminfo.
 *
 * Conventions
 *  - All tensors passed to kv_append / kv_attend are DEVICE pointers, F32.
 *  - Calls are ordered on the given CUDA stream (a cudaStream_t passed as
 *    void*; NULL = the legacy default stream).  No call blocks the host except
 *    kv_alloc, kv_free and the row import/export helpers.
 *  - Errors are negative return codes; the library never exits the process
 *    (the reference prints and calls exit(1), model.cpp:859-865).
 *  - One host thread drives one kv_ctx; the context's scratch is shared by
 *    its calls, so calls on one context must not overlap on the device.
 */
#ifndef KV_API_H
#define KV_API_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- return codes -------------------------------------------------------- */
#define KV_OK              0
#define KV_E_ARG          -1  /* bad argument or unsupported shape          */
#define KV_E_OOM          -2  /* device or host allocation failed           */
#define KV_E_RANGE        -3  /* row range outside [0, n_ctx) / batch limit */
#define KV_E_CUDA         -4  /* CUDA runtime error                         */
#define KV_E_COMM         -5  /* collective (NCCL) error                    */
#define KV_E_TIMEOUT      -6  /* a bounded device-side wait gave up         */
#define KV_E_STATE        -7  /* call order violated (attend w/o append)    */
#define KV_E_UNSUPPORTED  -8  /* feature not built / not available          */

/* ---- RoPE modes (ggml values, model.cpp:1395) ---------------------------- */
#define KV_ROPE_NORMAL 0      /* adjacent pairs (llama)                   */
#define KV_ROPE_NEOX   2      /* split halves (phi3 / qwen2 / qwen3)      */

typedef struct kv_ctx kv_ctx;

/*
 * Model attention parameters, the subset of `struct hparams` (model.h:63-95)
 * that the path reads, plus allocation and sharding options.
 */
typedef struct kv_config {
    int32_t n_layer;            /* hparams::n_layer                               */
    int32_t n_head;             /* hparams::n_head (query heads, whole model)     */
    int32_t n_head_kv;          /* hparams::n_head_kv                             */
    int32_t head_dim;           /* hparams::n_embd_head; 64, 96, 128 or 256 (256:
                                   whole-head RoPE)                             */
    int32_t n_rot;              /* hparams::n_rot (even, <= head_dim)             */
    int32_t rope_mode;          /* KV_ROPE_NORMAL (llama) / KV_ROPE_NEOX (others) */
    float   rope_base;          /* hparams::rope_freq_base                        */
    float   rope_freq_scale;    /* 1.0 for every reference architecture           */
    float   rope_attn_factor;   /* hparams::rope_attn_factor (mscale)             */
    float   rope_ext_factor;    /* 1.0 with phi3 LongRoPE, else 0 (model.cpp:1312)*/
    float   rope_beta_fast;     /* 32 with LongRoPE, else 0                       */
    float   rope_beta_slow;     /* 1 with LongRoPE, else 0                        */
    int32_t n_ctx_orig;         /* hparams::n_ctx_orig                            */
    const float *rope_freq_factors; /* HOST [n_rot/2] or NULL; copied by kv_alloc.
                                   phi3 rope_factors_short (model.cpp:555-557) or
                                   llama3 rope_freqs                             */
    int32_t qk_norm;            /* 1: hparams::has_qk_norm (qwen3): RMSNorm * gamma
                                   before RoPE.  2: dory's nGPT handling
                                   (dory.c:577-580, 646-649): after RoPE,
                                   rms_norm(x, rms_eps/head_dim) / sqrt(head_dim),
                                   Q then times q_norm_w [n_head][head_dim] (the
                                   squared learned scale); k_norm_w unused     */
    float   rms_eps;            /* hparams::rms_eps                               */
    int64_t n_ctx;              /* cache positions (<= 2^31); 0 = auto from free HBM */
    int64_t n_ctx_train;        /* auto-sizing clamp; 0 = 262144 cap              */
    int32_t longrope_clamp;     /* 1: auto-sizing also clamps to n_ctx_orig
                                   (phi3 with LongRoPE, model.cpp:1037-1039)     */
    int32_t n_batch_max;        /* max n_new per call; 0 = 512                    */
    int32_t device;             /* CUDA device ordinal; -1 = current device       */
    int32_t n_shards;           /* GPUs sharing the cache by KV head; 0/1 = one   */
    int32_t shard;              /* this context's shard index in [0, n_shards)    */
    const void *comm_id;        /* 128-byte id from kv_comm_unique_id() on shard 0,
                                   the same bytes on every shard; n_shards > 1    */
    int64_t ring_cells;         /* 0: linear cache, position p in row p.  > 0: a
                                   ring of ring_cells rows (dory.c:391-522), the
                                   token at position p in row p % ring_cells;
                                   n_ctx then bounds the positions (RoPE table)  */
    int32_t flash_attn;         /* 1: kv_attend (and kv_forward) take the flash-attn
                                   branch, as decode_session::use_flash_attn
                                   selects it (model.h:381-384); see
                                   KV_ATTN_FLASH at kv_attend_mask              */
    int32_t cache_type;         /* KV_CACHE_F16, or KV_CACHE_Q8: the cache in 8-bit
                                   codes (see kv_q8_cache), half the bytes       */
    int64_t cache_rows;         /* KV_CACHE_Q8: rows a layer holds (rounded up to a
                                   multiple of 32), 0 = n_ctx.  Fewer than n_ctx:
                                   kv_evict makes room                           */
    int32_t track_weights;      /* KV_CACHE_Q8: 1 = kv_attend accumulates each row's
                                   attention weight, which kv_evict goes by      */
} kv_config;

#define KV_CACHE_F16 0
#define KV_CACHE_Q8  1

/* Defaults: NEOX RoPE, base 10000, scale 1, attn factor 1, no YaRN, eps 1e-6,
 * n_ctx 0 (auto), n_batch_max 512, device -1, one shard, linear F16 cache.
 * Shape fields 0.
 *
 * 8-bit caches (cache_type KV_CACHE_Q8): the calls below are the same; kv_append
 * rotates and norms as it does for F16 and stores the F16 rows' codes, kv_attend
 * is kv_q8_attend's operator (queries rounded to F16, F32 out; the default and
 * the flash-attn branch differ only in a row without a visible key).  A layer's
 * positions have no gaps: kv_append refuses an n_past beyond the next one
 * (KV_E_RANGE).  One shard, no ring.
 *
 * Ring caches (ring_cells > 0; dory's sliding and global rings, one context
 * per ring size, per-loop slots as extra layers): kv_append's n_past is the
 * position of the first new token (RoPE and the cell p % ring_cells; n_new <=
 * ring_cells), and kv_attend attends over the min(ring_cells, n_past + n_new)
 * cells in use with dory_fill_attn_mask's visibility (dory.c:553-575: a cell
 * is visible to the query at p when its newest write is a real position <= p),
 * built on the device; kv_attend_mask takes the caller's mask over those cells
 * instead (mask_stride >= the cells in use). */
int kv_config_init(kv_config *cfg);

/* Bytes of the whole K+V cache at n_ctx positions, all layers and all shards:
 * exactly kv_cache_bytes() of the reference (model.cpp:869-885); a ring
 * configuration holds min(ring_cells, n_ctx) rows; an 8-bit one its codes,
 * scales and weights.  UINT64_MAX when the product does not fit 64 bits. */
uint64_t kv_cache_bytes(const kv_config *cfg, int64_t n_ctx);

/* Context auto-sizing rule of auto_n_ctx() (model.cpp:1002-1059) applied to
 * `free_bytes` of one GPU: (free - 384 MiB) * 0.8 / per-position bytes of this
 * shard (cache rows + RoPE table row), rounded down to a multiple of 64,
 * clamped to n_ctx_train (262144 if 0) and n_ctx_orig with longrope_clamp,
 * floor 512.  free_bytes <= 0 gives the reference's fallback, 4096. */
int64_t kv_auto_n_ctx(const kv_config *cfg, int64_t free_bytes);

/* Allocate the cache (+ RoPE table + scratch) on the configured device;
 * replaces init_kv_cache (model.cpp:821-867).  With cfg->n_ctx == 0 the size
 * comes from kv_auto_n_ctx(cudaMemGetInfo free).  With n_shards > 1 this
 * context owns KV heads [shard*n_head_kv/n_shards, (shard+1)*...) and the
 * matching query heads, and joins the collective identified by comm_id (every
 * shard must call kv_alloc concurrently, one process or thread per GPU).
 * Returns KV_OK, KV_E_ARG, KV_E_OOM, KV_E_CUDA or KV_E_COMM. */
int kv_alloc(const kv_config *cfg, kv_ctx **out);

/* Release everything kv_alloc acquired.  NULL is a no-op. */
int kv_free(kv_ctx *ctx);

/* Positions the cache holds (the n_ctx actually allocated). */
int kv_n_ctx(const kv_ctx *ctx, int64_t *n_ctx);

/*
 * Append n_new tokens' K and V rows at cache rows [n_past, n_past+n_new) of
 * `layer`, after QK-Norm (if cfg->qk_norm) and RoPE of K; also rotates Q into
 * the context for the following kv_attend.  Replaces model.cpp:1382-1414.
 *
 * q: token t's Q block (n_head*head_dim floats, heads outer) at q + t*q_stride;
 * k, v likewise with n_head_kv*head_dim floats.  For phi3's fused QKV output
 * (model.cpp:1088-1094) pass q = row, k = row + n_head*head_dim,
 * v = row + (n_head+n_head_kv)*head_dim and all three strides equal to the
 * fused row width.  q_norm_w / k_norm_w: [head_dim] gamma of this layer, or
 * NULL without QK-Norm.  Sharded contexts read only their own heads.
 * The F32 -> F16 cast rounds to nearest even; cache bytes equal the reference
 * CPU path's bit for bit.
 */
int kv_append(kv_ctx *ctx, int32_t layer, int64_t n_past, int32_t n_new,
              const float *q, int64_t q_stride,
              const float *k, int64_t k_stride,
              const float *v, int64_t v_stride,
              const float *q_norm_w, const float *k_norm_w,
              void *stream);

/*
 * kv_append with the QKV bias of qwen2-style layers (model.cpp:1099-1102,
 * ggml_add of attn_q/k/v.bias to the projections) added inside the append's
 * load: q_bias [n_head*head_dim], k_bias and v_bias [n_head_kv*head_dim], F32
 * device pointers of this layer, or NULL (no bias).  Each element is one
 * rounded F32 add before QK-Norm and RoPE, as ggml_add is.  kv_append is this
 * call with three NULL biases.
 */
int kv_append_bias(kv_ctx *ctx, int32_t layer, int64_t n_past, int32_t n_new,
                   const float *q, int64_t q_stride,
                   const float *k, int64_t k_stride,
                   const float *v, int64_t v_stride,
                   const float *q_norm_w, const float *k_norm_w,
                   const float *q_bias, const float *k_bias, const float *v_bias,
                   void *stream);

/*
 * Attention of the n_new tokens last appended to `layer` (same layer, n_past
 * and n_new as that kv_append) over cache rows [0, n_past+n_new) with the
 * causal mask k <= n_past+t (model.cpp:1579-1586) and scale 1/sqrt(head_dim).
 * out: [n_new][n_head*head_dim] F32, heads outer -- the layout of
 * `cur` after ggml_cont_2d at model.cpp:1444.  With n_shards > 1 every shard
 * receives the whole gathered output.  Only rows < n_past+n_new are read, so
 * rewinding n_past and overwriting rows is allowed (cmd_chat.cpp:749-764).
 */
int kv_attend(kv_ctx *ctx, int32_t layer, int64_t n_past, int32_t n_new,
              float *out, void *stream);

/* Mask element types and flags of kv_attend_mask. */
#define KV_MASK_F32    0   /* ggml_soft_max_ext's mask (model.cpp:1437)          */
#define KV_MASK_F16    1   /* the flash branch's ggml_cast mask (model.cpp:1431) */
#define KV_ATTN_FLASH  1u  /* the ggml_flash_attn_ext branch (model.cpp:1426-1434) */

/*
 * kv_attend with the reference's explicit additive mask in place of the
 * implicit causal one, and the choice of the reference's two attention
 * branches (decode_session::use_flash_attn, model.h:381-384).  Same call order
 * and output as kv_attend.
 *
 * mask: DEVICE pointer to n_new rows of at least n_past+n_new elements,
 * mask_stride elements apart (the [n_kv, n_new] mask model.cpp:1579-1586
 * builds, rows padded as ggml pads them), F32 (KV_MASK_F32) or F16
 * (KV_MASK_F16); the score of token t and key k is dot*scale + mask[t][k], so
 * -inf removes the key.  NULL keeps the implicit causal mask.  Rows starting on
 * 16-byte boundaries are read with vector loads.
 * flags: 0 = the default branch (ggml_soft_max_ext then ggml_mul_mat: the
 * normalised weights rounded to F16); KV_ATTN_FLASH = the ggml_flash_attn_ext
 * branch: the weights exp(s - max) are not normalised before the F16 rounding
 * (the output is divided by their sum), and a row whose keys are all masked
 * gives 0 (the default branch gives NaN, as ggml's soft_max of an all -inf
 * row).  The flash branch's output layout [head_dim, n_head, n_new] is the
 * same memory order as `out` here.
 * Returns KV_OK, KV_E_ARG (unknown type or flag, mask_stride < n_past+n_new)
 * or the codes of kv_attend.
 */
int kv_attend_mask(kv_ctx *ctx, int32_t layer, int64_t n_past, int32_t n_new,
                   const void *mask, int32_t mask_type, int64_t mask_stride,
                   uint32_t flags, float *out, void *stream);

/*
 * One step of the path over every layer: for layer l in [0, n_layer),
 * kv_append then kv_attend with inputs at q + l*in_layer_stride (likewise k,
 * v), gammas at q_norm_w + l*norm_layer_stride, output at
 * out + l*out_layer_stride.  The per-layer loop of forward_step
 * (model.cpp:1318, 1496-1597) restricted to this path, driven from C++.  On an
 * 8-bit context a layer without room (KV_E_RANGE) is found before the first
 * layer's work, so the call can be made again after kv_evict.
 */
int kv_forward(kv_ctx *ctx, int64_t n_past, int32_t n_new,
               const float *q, int64_t q_stride,
               const float *k, int64_t k_stride,
               const float *v, int64_t v_stride, int64_t in_layer_stride,
               const float *q_norm_w, const float *k_norm_w, int64_t norm_layer_stride,
               float *out, int64_t out_layer_stride, void *stream);

/*
 * Decode attention that allocates nothing.  No counterpart in the reference:
 * it exists for callers that cannot call cudaMalloc -- a host framework that
 * owns and plans all device memory up front (ggml's graph allocator, a serving
 * engine that reserves HBM for its own pool) and runs this op as a callback in
 * the middle of its compute, where an allocation would fail for lack of free
 * memory or stall the device.  Such a caller cannot hold a kv_ctx (kv_alloc
 * allocates), so it passes its own cache and buffers:
 *   k_cache, v_cache: one layer's cache, [rows][n_head_kv][head_dim] F16,
 *                     16-byte aligned; rows [0, n_kv) are attended, the new
 *                     token's K/V already written at row n_kv-1;
 *   q:   the new token's rotated query, [n_head][head_dim] F32 (device);
 *   out: [n_head*head_dim] F32 (device), the layout kv_attend writes.
 * It runs kv_attend's decode attention kernel (its default branch -- not the
 * flash-attn one -- over a plain grid, launched cooperatively so the driver
 * starts it only with all its CTAs resident).  Its scratch is a fixed 16 MiB
 * array built into the library (held by every GPU that loads it until exit);
 * a call needs about 32 bytes of it per (KV head, key) for scores -- about
 * 56k keys with 8 KV heads, 14k with 32 -- and returns KV_E_RANGE, with
 * kv_last_error() saying so, when the shape does not fit.  The first call on
 * a device looks up the array's device address and sets up the kernel, so
 * make it before any stream capture; a cudaDeviceReset() invalidates that
 * set-up for the rest of the process.  Calls share the array: calls that
 * overlap on the GPU race and must be serialised.
 */
int kv_attend_decode_noalloc(const uint16_t *k_cache, const uint16_t *v_cache,
                             int32_t n_head, int32_t n_head_kv, int32_t head_dim, int64_t n_kv,
                             const float *q, float *out, void *stream);

/*
 * Evict rows of `layer` of an 8-bit context with track_weights: each KV head
 * keeps the layer's last `recent` rows and the heaviest others, `keep` in all
 * (kv_q8_evict; keep at most the rows in use).  Positions are not renumbered:
 * the kept keys stay rotated as they are, the next kv_append is again at the
 * next position, n_past, and kv_attend attends over the rows that are left.
 * The weight is what every kv_attend since a row's kv_append gave it, those of
 * tokens rewound since, and of calls made twice, among them.
 * Every layer is evicted by its own call.  Rewinding n_past is possible by up
 * to `recent` tokens, as far as an earlier eviction allowed it (KV_E_RANGE
 * beyond), or to 0.  kept: DEVICE int32
 * [n_head_kv][keep], each head's kept rows (their numbers before the call), or
 * NULL.  The layer's buffers change places with a spare set, so a stream that is
 * being captured is refused (KV_E_STATE), and a graph captured before must not
 * be replayed after.
 */
int kv_evict(kv_ctx *ctx, int32_t layer, int64_t keep, int64_t recent, int32_t *kept, void *stream);

/* Rows of `layer` in use, and rows it holds (either may be NULL). */
int kv_layer_rows(const kv_ctx *ctx, int32_t layer, int64_t *used, int64_t *capacity);

/* ---- the cache in 8 bits -------------------------------------------------- */
/*
 * One layer's K and V in 8-bit codes with one scale for each KV head and block
 * of KV_Q8_BLOCK consecutive rows: half the bytes an attention call streams
 * and half the memory of the F16 cache.  No counterpart in the reference,
 * whose cache is F16.  The calls below work on the caller's buffers and
 * allocate nothing, as kv_attend_decode_noalloc does.
 *
 *   code c of row i, block b = i / KV_Q8_BLOCK, stands for c * scale[h][b];
 *   scale = 2^e with the smallest e in [-24, 9] at which the block's largest
 *   magnitude rounds to a code <= 127 (e = 9 saturates there): a power of two,
 *   so every value is an exact F16, and a row that moves to another block of
 *   the same scale keeps its codes.  A value is first rounded to F16, as the
 *   F16 cache would hold it.  What is not finite then (inf, NaN) has code -128,
 *   which reads back as NaN, and its block's scale is NaN (the exponent kept in
 *   the low byte): attention takes every row of such a block as NaN.
 *
 * What that costs: a value is off by up to half its block's scale, scale /
 * sqrt(12) in the mean, and 32 rows of a head share one scale, set by their largest
 * magnitude.  With queries and values of size 1 an output is off by about
 * sqrt(sk^2 + sv^2) / sqrt(12) of its size, sk and sv the scales: 1.7 % with normally
 * distributed rows of 128, 3.8 % where four channels of K lie 8 deviations off the
 * others, 14 % where two lie 30 off (2048 keys).  K with channels far larger than
 * the rest is what this format is worst at.
 *
 * All pointers are DEVICE pointers on the current device, k and v 16-byte
 * aligned; rows is a multiple of KV_Q8_BLOCK, at most 2^31 - 32.  head_dim: 64,
 * 96, 128 or 256.  n_head_kv: at most 1024.
 */
#define KV_Q8_BLOCK 32

typedef struct kv_q8_cache {
    int8_t *k, *v;              /* [n_head_kv][rows][head_dim] codes            */
    float *k_scale, *v_scale;   /* [n_head_kv][rows / KV_Q8_BLOCK]              */
    float *weight;              /* [n_head_kv][rows] accumulated attention weight,
                                   or NULL: none is kept                        */
    int64_t rows;
    int32_t n_head_kv, head_dim;
} kv_q8_cache;

/* Element types of the calls below (those of the mask: KV_MASK_F32, KV_MASK_F16). */
#define KV_F32 0
#define KV_F16 1

/*
 * Store n_new rows (rotated and normed by the caller, as kv_append writes them)
 * at cache rows [row0, row0+n_new): token t's K heads at k + t*k_stride
 * elements, [n_head_kv][head_dim], V likewise.  Rows [0, row0) are kept; the
 * first block's rows before row0 get the block's new scale where that changed
 * (a growing scale rounds their codes once more).  Rows behind row0+n_new are
 * not written, but a block's scale is that of its rows before row0+n_new: store
 * them again before they are read.  The new rows' weights become 0.
 * Returns KV_OK, KV_E_ARG, KV_E_RANGE (rows outside the cache) or KV_E_CUDA.
 */
int kv_q8_store(const kv_q8_cache *cache, int64_t row0, int32_t n_new, const void *k, int64_t k_stride,
                const void *v, int64_t v_stride, int32_t type, void *stream);

/*
 * The values of rows [row0, row0+n) as F16 (exact) or F32: row i's heads at
 * k_out + (i-row0)*stride elements, [n_head_kv][head_dim], V likewise; either
 * may be NULL.
 */
int kv_q8_load(const kv_q8_cache *cache, int64_t row0, int64_t n, void *k_out, void *v_out, int64_t stride,
               int32_t type, void *stream);

/* Bytes of workspace kv_q8_attend needs for these sizes (0: bad arguments).  It
 * grows with n_past and n_new: ask once for the largest of both.  The contents
 * need no preparation; calls that overlap on the device need one each (and on
 * a cache that keeps weights no two calls may overlap). */
uint64_t kv_q8_attend_workspace(const kv_q8_cache *cache, int32_t n_head, int64_t n_past, int32_t n_new);

/*
 * Attention of n_new tokens, whose rows [n_past, n_past+n_new) are stored, over
 * rows [0, n_past+n_new) with scale 1/sqrt(head_dim): kv_attend's operator over
 * the 8-bit cache.  q: token t's rotated query heads at q + t*q_stride elements,
 * [n_head][head_dim], F32 (rounded to F16 as kv_attend does) or F16.  out: token
 * t's heads at out + t*out_stride, F32 or F16 (q_type / out_type).
 * mask, mask_type, mask_stride, flags: as kv_attend_mask (NULL: causal; the
 * flags change only a row without a visible key: NaN, or 0 with KV_ATTN_FLASH).
 * A key masked with -inf does not enter the row, whatever its block holds.
 * Scores may be of any finite size with at most 16 query rows a KV head (n_new *
 * n_head / n_head_kv), or with a mask; else one past 10^7 (or below -10^7) may
 * make its row NaN, as one that is not finite does.
 * With cache->weight, weight[h][i] of every attended row i grows by the softmax
 * weights that the n_new tokens' query heads of KV head h gave it; a query row
 * whose softmax is not finite (no visible key, NaN or inf scores) adds nothing.
 * The weights are a sum over calls: a call made twice for the same rows, a
 * replayed graph, and draft tokens that are rewound afterwards have all left
 * theirs in the rows that stay (kv_q8_store sets only its own rows' to 0).
 * Results do not depend on timing (no atomics).  On their way to V the softmax
 * weights are rounded to 22 bits with up to 4 query rows a KV head (n_new * n_head
 * / n_head_kv) and to F16 with more, as kv_attend rounds them, so a token's bits
 * alone and among others differ.
 * workspace: 256-byte aligned device memory of at least kv_q8_attend_workspace
 * bytes.  Returns KV_OK, KV_E_ARG, KV_E_RANGE (rows outside the cache, n_new or
 * workspace too small or large) or KV_E_CUDA.  n_new: at most 65535.
 */
int kv_q8_attend(const kv_q8_cache *cache, int32_t n_head, int64_t n_past, int32_t n_new,
                 const void *q, int64_t q_stride, int32_t q_type,
                 const void *mask, int32_t mask_type, int64_t mask_stride, uint32_t flags,
                 void *out, int64_t out_stride, int32_t out_type,
                 void *workspace, uint64_t workspace_bytes, void *stream);

/* Deferred device-side errors of kv_q8_attend on the current device, as
 * kv_status: waits for `stream`, then returns KV_E_TIMEOUT (and clears the
 * record) if a bounded wait inside one of its kernels expired since the last
 * check (the outputs of that call are not valid, and its softmax weights are
 * added to none of the rows or, where the wait was in the weights' own pass, to
 * some), else KV_OK.  One record a device, for all calls of kv_q8_attend there; a kv_ctx has its own, which
 * kv_status reads. */
int kv_q8_status(void *stream);

/*
 * Evict rows by accumulated attention weight.  Of the first n_rows rows of
 * `src`, each KV head keeps its last `recent` ones and, of those before, the
 * keep-recent of largest weight (equal weights: the lower row; a NaN weight
 * counts as the largest), in ascending order, at rows [0, keep) of `dst`: their
 * values at the new blocks' scales, their weights (where dst has them), and
 * their rows in src in kept, int32 [n_head_kv][keep].  dst is another cache of
 * the same n_head_kv and head_dim; none of its buffers may overlap one of
 * src's.  0 <= recent <= keep <= n_rows, keep >= 1.
 */
int kv_q8_evict(const kv_q8_cache *src, int64_t n_rows, int64_t keep, int64_t recent,
                const kv_q8_cache *dst, int32_t *kept, void *stream);

/* Copy cache rows [row0, row0+nrows) of K (which = 0) or V (which = 1) of
 * `layer` to / from host memory in the reference layout [row][head][dim] F16
 * (this context's heads only; an 8-bit cache's values, exact in F16, or stored
 * as kv_q8_store stores them: the rows in use before row0 in its block, and
 * those behind in the last block, are stored again at the block's scale).
 * Synchronous.  Used for checking, for the reference's /save-/load style
 * rebuilds and for tests.  On an 8-bit context rows are counted as
 * kv_layer_rows counts them, and imported rows are in use from then on: those
 * that were not have weight 0, and zeros in the other of K and V (and, where
 * row0 lies behind the rows in use, in the rows between) until that is imported
 * too.  An import does not undo an eviction: positions stay as far from rows as
 * kv_evict left them, so a session that was saved whole goes into a context of
 * its own, or one that began again at n_past 0. */
int kv_export_rows(kv_ctx *ctx, int32_t layer, int32_t which, int64_t row0,
                   int64_t nrows, uint16_t *host_dst);
int kv_import_rows(kv_ctx *ctx, int32_t layer, int32_t which, int64_t row0,
                   int64_t nrows, const uint16_t *host_src);

/* Shard geometry of a context: first global query head, query heads, first
 * global KV head, KV heads. */
int kv_shard_info(const kv_ctx *ctx, int32_t *q_head0, int32_t *n_q_heads,
                  int32_t *kv_head0, int32_t *n_kv_heads);

/* 128-byte identifier for a new collective; call on shard 0 and hand the
 * bytes to every shard's kv_config.comm_id.  KV_E_UNSUPPORTED when NCCL
 * (libnccl.so.2) cannot be loaded. */
int kv_comm_unique_id(void *id_out);

/* Deferred device-side errors: waits for `stream`, then returns KV_E_TIMEOUT
 * (and clears the record) if a bounded wait inside one of this context's
 * kernels expired since the last check -- the outputs of that call are not
 * valid (and its weights, on an 8-bit context, as kv_q8_status says) -- else
 * KV_OK.  The context stays usable either way. */
int kv_status(kv_ctx *ctx, void *stream);

const char *kv_strerror(int code);
/* Detail of the last failing call on this host thread ("" if none). */
const char *kv_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* KV_API_H */
