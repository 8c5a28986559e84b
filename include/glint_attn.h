/*
 * glint_attn.h -- C ABI of the MI355X (gfx950) attention path for Glint.
 *
 * This library replaces the attention step of Glint's GPU backend and its
 * CPU flash-attention fallback:
 *   - GpuBackend::attention / attention_resident   src/backend/gpu.rs:266-397, :860-992
 *   - GpuBackend::create_kv_cache / GpuKvCache      src/backend/gpu.rs:1039-1104
 *   - KvStore::write / export_raw / import_raw      src/cache/mod.rs:24-109
 *   - PagePool page recycle and copy-on-write       src/cache/paged.rs:79-82, :433-444
 *   - attn_heads_cpu over a batch (decode)          src/transformer/forward.rs:1468-1502
 *   - prefill attention loop                        src/transformer/forward.rs:927-958
 * and, beside it on a decode step, RoPE (src/tensor/ops.rs:212-245), the
 * Q8_0 weight matvec (src/tensor/quantized.rs:247-346, :587-610), the 4-bit
 * one, the append of rotated rows to a storage and the norms between blocks.
 * The numerics follow flash_attn_1d_ext (src/tensor/flash.rs:46-124).
 *
 * Conventions (the same as Glint's outbound C API, include/glint.h:21-35):
 *   - Every function returns an int status: GLA_OK (0) or a negative code.
 *     gla_last_error() returns a thread-local message for the last failure on
 *     the calling thread. No C++ exception crosses the boundary.
 *   - Handles are not thread-safe; use one gla_ctx per thread or lock.
 *   - "Device" pointers are HIP device addresses on the context's device;
 *     "host" pointers are ordinary memory borrowed for the call only.
 *   - Device-pointer entry points are asynchronous on the context's stream;
 *     gla_sync() waits for them. Host-pointer entry points return after the
 *     results are in host memory.
 *   - Unsupported shapes return GLA_ERR_INVALID so the caller can take its
 *     CPU path, as it does for the wgpu MAX_SEQ guard (src/backend/gpu.rs:277-282).
 *
 * Supported shapes: head_dim in {64, 128, 256}; any n_heads that is a
 * multiple of n_kv_heads; any context length (no MAX_SEQ limit).
 */
#ifndef GLINT_ATTN_H
#define GLINT_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. The GPU ones correspond to GlintError (src/error.rs:41-52, :78-82). */
#define GLA_OK 0
#define GLA_ERR_NO_DEVICE (-1)      /* GlintError::GpuAdapterNotFound */
#define GLA_ERR_DEVICE (-2)         /* GlintError::GpuDeviceError */
#define GLA_ERR_BUFFER (-3)         /* GlintError::GpuBufferError (alloc / copy) */
#define GLA_ERR_KERNEL (-4)         /* GlintError::GpuShaderError (launch) */
#define GLA_ERR_INVALID (-5)        /* bad argument or unsupported shape */
#define GLA_ERR_POOL_EXHAUSTED (-6) /* GlintError::KvPagePoolExhausted */

/* Positions per page -- src/cache/paged.rs:55 PAGE_SIZE. */
#define GLA_PAGE_SIZE 16

/* KV element formats: KvCache / PagedKvCache (f32) and KvCacheQ8 (Q8_0,
 * 32-element blocks with one f16 scale, src/cache/mod.rs:263-315). */
typedef enum gla_kv_dtype { GLA_KV_F32 = 0, GLA_KV_Q8_0 = 1 } gla_kv_dtype;

/* Arithmetic of the prefill matrix products. */
typedef enum gla_precision {
    GLA_PREC_F32 = 0, /* fp32: every operand as two f16 pieces (22 bits at any
                         magnitude), three f16 MFMAs a product, fp32
                         accumulation; closer to 64 bits than fp32 MFMAs. A
                         query row's bits follow from the row and the keys it
                         attends alone. */
    GLA_PREC_BF16 = 1 /* bf16-rounded Q/K/P/V inputs, fp32-accumulate MFMA */
} gla_precision;

typedef struct gla_ctx gla_ctx;
typedef struct gla_kv gla_kv;

/* ---- context ------------------------------------------------------------ */

/* Thread-local message of the last failed call on this thread ("" if none).
 * Replaces glint_last_error (include/glint.h, src/ffi/mod.rs:64). */
const char *gla_last_error(void);

/* Open `device`. Returns GLA_ERR_NO_DEVICE when no HIP device is present,
 * the condition GpuBackend::new reports as GpuAdapterNotFound
 * (src/backend/gpu.rs:44-56); the caller then stays on its CPU path. */
int gla_create(int device, gla_ctx **out);
/* Frees the context and the device memory of every cache, pool, weight set
 * and rotary plan created on it; their handles must still be released
 * (gla_kv_destroy, gla_q8w_destroy, gla_q4w_destroy, gla_rope_plan_destroy),
 * which then frees only the handle, and any other use of them fails with
 * GLA_ERR_INVALID. */
int gla_destroy(gla_ctx *ctx);

/* Run subsequent work on `hip_stream` (a hipStream_t); NULL restores the
 * context's own stream. Each stream the context has launched work on has
 * its own device scratch (decode split partials, prefill tile images,
 * matvec activation pieces), so calls queued on different streams at once
 * never share it and may overlap; calls on one stream run in order as usual.
 * A graph uses the scratch of the stream it was captured on: graphs of one
 * stream are replayed one after another, wherever they are launched, and one
 * that is launched on another stream never beside the first one's own calls
 * (they would share partial sums, pieces and counters): wait in between.
 * That scratch is held until gla_destroy or gla_release_stream. The stream
 * must outlive its use by the context: switch away from it (or release it)
 * before destroying it. The context itself is not thread-safe: switch
 * streams from one thread. */
int gla_set_stream(gla_ctx *ctx, void *hip_stream);
/* The hipStream_t work is enqueued on. */
void *gla_get_stream(gla_ctx *ctx);
/* Free the device scratch the context keeps for `hip_stream` (split
 * partials, tile images, matvec pieces), after waiting for that stream.
 * Scratch is otherwise held per stream until gla_destroy, so a caller that
 * makes a stream per request calls this before destroying each stream. If
 * `hip_stream` is the current stream, the context first returns to its own
 * stream. Graphs captured on `hip_stream` must not be replayed afterwards.
 * Buffers that a stream's scratch outgrew stay allocated until gla_destroy
 * (earlier graphs may address them). Releasing a stream the context never
 * used is a no-op. */
int gla_release_stream(gla_ctx *ctx, void *hip_stream);
/* Wait for all work enqueued on the context's stream. */
int gla_sync(gla_ctx *ctx);
/* Number of compute units of the context's device (0 on error). */
int gla_device_cu_count(gla_ctx *ctx);


/* ---- device memory (for device-resident q / out / tables) --------------- */

int gla_dev_alloc(gla_ctx *ctx, size_t bytes, void **out);
int gla_dev_free(gla_ctx *ctx, void *ptr);
/* Host -> device; returns once `src` may be reused. */
int gla_memcpy_htod(gla_ctx *ctx, void *dst_dev, const void *src_host, size_t bytes);
/* Device -> host; waits for the context's stream first. */
int gla_memcpy_dtoh(gla_ctx *ctx, void *dst_host, const void *src_dev, size_t bytes);

/* ---- KV storage ---------------------------------------------------------- */

/* Contiguous caches for n_seqs sequences: each holds max_seq_len positions of
 * every layer, like KvCache::new / KvCacheQ8::new (src/cache/mod.rs:127-140,
 * :288-294) and GpuBackend::create_kv_cache (src/backend/gpu.rs:1060-1104).
 * Storage is zero-initialised. */
int gla_kv_cache_create(gla_ctx *ctx, gla_kv_dtype dtype, int n_seqs, int n_layers, int max_seq_len,
                        int n_kv_heads, int head_dim, gla_kv **out);

/* A pool of capacity_pages pages; a page holds GLA_PAGE_SIZE positions of K
 * and V of one layer and has no layer identity, like PagePool::preallocated
 * (src/cache/paged.rs:176-189). Page ids run 0 .. capacity_pages-1; the caller
 * keeps the page tables and reference counts (PagedKvCache's table[layer][page],
 * src/cache/paged.rs:254-260). Storage is zero-initialised. */
int gla_pool_create(gla_ctx *ctx, gla_kv_dtype dtype, int n_kv_heads, int head_dim, int capacity_pages,
                    gla_kv **out);

int gla_kv_destroy(gla_kv *kv);

/* Row id of (seq, layer, pos) in a contiguous cache; row ids of a pool are
 * page * GLA_PAGE_SIZE + slot. Returns -1 on a bad argument. */
int64_t gla_kv_row_id(const gla_kv *kv, int seq, int layer, int pos);

/* Write K and V rows (kv_dim = n_kv_heads * head_dim floats each) -- the
 * KvStore::write analogue (src/cache/mod.rs:166-177, :374-388,
 * src/cache/paged.rs:467-490). Q8_0 storage quantises on write with the
 * rules of KvCacheQ8::quantize_into (src/cache/mod.rs:296-315), bit-exactly.
 * Device pointers; asynchronous. rows: int64[n_rows]; k, v: [n_rows][kv_dim].
 * The rows are written in parallel: where ids are repeated within one call
 * every stored value is one of theirs, which one is unspecified and may differ
 * from value to value (a Q8_0 quant may lie beside another row's scale): repeat
 * none that is read later. Ids outside the storage are skipped on the device. */
int gla_kv_write_rows(gla_ctx *ctx, gla_kv *kv, const int64_t *rows_dev, const float *k_dev,
                      const float *v_dev, int n_rows);
/* The same with host pointers; returns when the rows are written. */
int gla_kv_write_rows_host(gla_ctx *ctx, gla_kv *kv, const int64_t *rows, const float *k, const float *v,
                           int n_rows);

/* Read rows back as the f32 values the storage holds of them (Q8_0: quant
 * times its block's f16 scale): the inverse of gla_kv_write_rows, for rows
 * that move to another storage or are rotated to other positions. Device
 * pointers, k and v 16-byte aligned; asynchronous. rows: int64[n_rows]; k, v:
 * [n_rows][kv_dim]. The outputs of ids outside the storage are left as they were. */
int gla_kv_read_rows(gla_ctx *ctx, const gla_kv *kv, const int64_t *rows_dev, float *k_dev, float *v_dev,
                     int n_rows);

/* Export rows as the bytes KvStore::export_raw produces for them
 * (src/cache/mod.rs:68-84, :219-241, :390-395): f32 rows are kv_dim native
 * floats; Q8_0 rows are ceil(kv_dim/32) blocks of [f16 scale LE][32 x i8].
 * Host pointers; k_out and v_out receive n_rows * row_bytes each. */
int gla_kv_export_rows_host(gla_ctx *ctx, const gla_kv *kv, const int64_t *rows, int n_rows, uint8_t *k_out,
                            uint8_t *v_out);
/* Inverse of export (KvStore::import_raw, src/cache/mod.rs:397-422):
 * stores the bytes as they are (Q8_0 blocks are not re-quantised). */
int gla_kv_import_rows_host(gla_ctx *ctx, gla_kv *kv, const int64_t *rows, int n_rows, const uint8_t *k_in,
                            const uint8_t *v_in);
/* Bytes one exported K (or V) row occupies. */
int64_t gla_kv_row_bytes(const gla_kv *kv);

/* Copy-on-write of a shared page (src/cache/paged.rs:433-444) and the
 * recycled-page wipe (PageBuf::reset, src/cache/paged.rs:79-82). Pools only;
 * asynchronous. */
int gla_pool_copy_page(gla_ctx *ctx, gla_kv *pool, int src_page, int dst_page);
int gla_pool_zero_page(gla_ctx *ctx, gla_kv *pool, int page);

/* ---- attention ----------------------------------------------------------- */

/* window_start of src/transformer/forward.rs:574-581: 0 on odd layers when
 * `alternating` (Gemma-2), else max(0, pos - sliding_window + 1) when
 * sliding_window > 0, else 0. attend_len is then pos + 1 - window_start. */
long gla_window_start(long pos, long sliding_window, int alternating, int layer);

/* Batched single-token decode: for every sequence b and q-head h,
 *   out[b][h] = softmax_j(cap(q[b][h] . K[j] * scale)) . V[j]
 * over positions j in [kv_start[b], kv_start[b] + kv_len[b]) of the sequence's
 * KV, K/V head h / (n_heads / n_kv_heads), cap(s) = softcap * tanh(s / softcap)
 * when softcap > 0 -- flash_attn_1d_ext per head (src/tensor/flash.rs:46-124)
 * as attn_heads_cpu calls it (src/transformer/forward.rs:240-270). kv_len 0
 * gives a zero output, as the reference's pre-zeroed buffer does. Non-finite
 * data behaves as there: a NaN reaching a head's weights or sums makes the
 * head's output NaN (the reference leaves such sums unnormalised,
 * flash.rs:118-123), and an infinite value under a non-zero weight gives
 * +-inf in its dimension.
 *
 * Out-of-range indices. The reference panics on a position or page id
 * outside the storage (Vec indexing in PagedKvCache::read_k_head,
 * src/cache/paged.rs:453-465; the write/truncate bounds of
 * src/cache/mod.rs:167-171, :186-190). Here:
 *   - with the host copies (kv_start_host / kv_len_host), every window is
 *     checked on the host before anything is launched: kv_start < 0,
 *     kv_len < 0, kv_len > max_kv_len, or kv_start + kv_len past the
 *     storage (the cache's max_seq; a pool's page_table_stride * 16
 *     positions) returns GLA_ERR_INVALID and the next call works;
 *   - the device arrays themselves are not read by the host. The kernels
 *     clamp every index they derive from them into the storage (positions
 *     to [0, storage positions), seq_slot to [0, n_seqs of the cache), page
 *     ids to [0, pages of the pool)), so a malformed device length, slot or
 *     page-table entry gives attention over the clamped positions and
 *     GLA_OK, never an access outside the storage. */
typedef struct gla_decode_args {
    const gla_kv *kv;          /* contiguous cache or pool */
    int layer;                 /* contiguous caches: layer to read; ignored for pools */
    int n_seqs;                /* batch size B */
    const int32_t *seq_slot;   /* caches: device int32[B], cache sequence read by batch row b
                                  (NULL: row b reads sequence b) */
    const int32_t *page_table; /* pools: device int32[B][page_table_stride], the physical page
                                  of each logical page pos / GLA_PAGE_SIZE (this layer's table) */
    int page_table_stride;
    const int32_t *kv_start; /* device int32[B]: window_start */
    const int32_t *kv_len;   /* device int32[B]: attend_len (>= 0) */
    int max_kv_len;          /* host: >= every kv_len[b] (sizes the launch) */
    int n_heads;
    float scale;   /* query_pre_attn_scalar or 1/sqrt(head_dim) (forward.rs:583-585) */
    float softcap; /* attn_logit_softcapping; <= 0 means none */
    const float *q; /* device [B][n_heads][head_dim] */
    float *out;     /* device [B][n_heads][head_dim] */
    /* Optional host copies of kv_start / kv_len: both NULL, or both int32[B]
     * holding the values of the device arrays. Read during the call only, to
     * size the launch to the batch's real lengths (the engine keeps every
     * sequence's position on the host, src/transformer/forward.rs:1468-1507,
     * so passing them is free); without them the launch is sized for
     * max_kv_len. */
    const int32_t *kv_start_host;
    const int32_t *kv_len_host;
} gla_decode_args;

int gla_decode(gla_ctx *ctx, const gla_decode_args *args);

/* Device scratch gla_decode_noalloc may use, in bytes (one array per GPU). */
#define GLA_DECODE_NOALLOC_SCRATCH_BYTES (16u << 20)
/* (sequence, KV head, head group) units an f32-storage gla_decode_noalloc
 * call may hold (arrival counters of the short-window merge; one array per
 * GPU). Never the tighter limit: a unit that counts arrivals has at least
 * two split partials of at least 384 bytes each, so the partial scratch
 * refuses a call before it reaches 21,846 such units. */
#define GLA_DECODE_NOALLOC_UNITS 65536

/* gla_decode that allocates nothing. It has no counterpart in the reference:
 * it is for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc). Same
 * arguments, kernels and bit-identical results as gla_decode; the split
 * partials live in a static device array of GLA_DECODE_NOALLOC_SCRATCH_BYTES
 * that each GPU the library runs on holds until the process ends (resolved
 * once per device by gla_create). A call whose partials need more returns
 * GLA_ERR_INVALID before anything is launched. The capacity depends on the
 * storage: at Llama-3-8B heads (32/8, d128) and 8,192 positions per
 * sequence, Q8_0 storage takes up to 192 sequences per call (B=64 needs
 * 5.3 MiB), f32 storage up to 29 (f32 splits are shorter: 33 partials per
 * KV head against 5). Every call on one GPU shares that GPU's array: calls
 * that overlap on one GPU (two streams or two contexts) race. Nothing in it
 * needs clearing: a call writes every partial it reads. f32 windows of at
 * most 65 pages (33 at head groups of over 512 floats) merge their splits in
 * the last workgroup to finish and count arrivals in a second static array of GLA_DECODE_NOALLOC_UNITS counters
 * (zero when the library loads, left at zero by every call); a call with
 * more (sequence, KV head, head group) units returns GLA_ERR_INVALID. */
int gla_decode_noalloc(gla_ctx *ctx, const gla_decode_args *args);

/* Batched causal prefill: query row r of sequence b sits at absolute
 * position pos_offset[b] + (r - q_start[b]) and attends positions
 * [w, that position] of the sequence's KV, w = max(0, pos - sliding_window + 1)
 * when sliding_window > 0 else 0 -- the loop of src/transformer/forward.rs:927-958
 * (pass sliding_window = 0 for a global layer of an alternating model). The
 * K/V of every attended position must already be written, as the reference
 * writes the chunk before attending (forward.rs:874-877).
 *
 * Out-of-range indices, as for gla_decode: the attended key positions are
 * clamped into the storage (a pos_offset past it attends the stored
 * positions only; a negative one attends none of its own) and seq_slot and
 * page-table entries into the cache or pool, so a malformed device value
 * gives clamped attention and GLA_OK where the reference would panic. The
 * query rows q_start[b] .. q_start[b+1]-1 index q and out, whose size the
 * library is not told: they must lie inside those buffers. */
typedef struct gla_prefill_args {
    const gla_kv *kv;
    int layer;
    int n_seqs;
    const int32_t *seq_slot;   /* caches: device int32[B] or NULL */
    const int32_t *page_table; /* pools: device int32[B][page_table_stride] */
    int page_table_stride;
    const int32_t *q_start;    /* device int32[B + 1]: query rows of b are q_start[b] .. q_start[b+1]-1 */
    const int32_t *pos_offset; /* device int32[B] */
    int max_q_len;             /* host: >= every q_start[b+1] - q_start[b] */
    int n_heads;
    float scale;
    float softcap;          /* <= 0: none */
    int sliding_window;     /* <= 0: none */
    gla_precision precision;
    const float *q; /* device [total_rows][n_heads][head_dim] */
    float *out;     /* device [total_rows][n_heads][head_dim] */
} gla_prefill_args;

int gla_prefill(gla_ctx *ctx, const gla_prefill_args *args);

/* ---- contexts that keep, or share, their beginning ----------------------- */

/* gla_decode whose rows also see the first n_sinks positions of their sequence,
 * where a window has left them behind: row b attends the positions
 * j < kv_start[b] + kv_len[b] with j >= kv_start[b] or j < n_sinks. kv_len,
 * max_kv_len and the host copies are the window's alone, as in gla_decode; a row
 * with kv_len 0 attends nothing (a zero output). n_sinks 0 is gla_decode; below 0
 * is refused. What gla_decode says of indices, non-finite data, host copies and
 * captures holds here. A row's bits follow from its own window and n_sinks. */
int gla_decode_sinks(gla_ctx *ctx, const gla_decode_args *args, int n_sinks);

/* gla_prefill whose rows also see the first n_sinks positions: the row at position
 * p attends the positions j <= p with j > p - sliding_window or j < n_sinks (all
 * of them without a window). n_sinks 0 is gla_prefill; below 0 is refused. */
int gla_prefill_sinks(gla_ctx *ctx, const gla_prefill_args *args, int n_sinks);

/* gla_decode of a batch whose neighbouring rows begin with the same positions: the
 * sequences that a prefix cache gave the same pages. Rows group_start[g] ..
 * group_start[g+1]-1 hold the same K and V at the positions before prefix_len[g];
 * those of the pages that lie wholly before it are read once for the group, through
 * its first row's pages (the table's row, or the cache's sequence), and multiplied
 * with the queries of all its rows as one matrix product, or by every row for itself
 * where the bounds, or the host copies, say that this is faster; what the copies show
 * exactly the bounds can only guess, and bounds far above what comes make a call slower.
 * Windows may begin or end inside the prefix or behind it: pages that no row sees are not
 * read. Rows in no group share nothing. The results are gla_decode's but for rounding,
 * which depends on the groups, the bounds and the copies: not bit-identical to it, nor
 * from one grouping to another.
 *
 * Values that the host does not see are clamped into the batch and the storage as
 * gla_decode's are: group starts that fall, or pages that differ where they are said
 * to be the same, give wrong rows and GLA_OK, never an access outside the buffers.
 * With the host copies they are checked before anything is launched
 * (GLA_ERR_INVALID). Allocates scratch of the stream as gla_decode does: call it once
 * before capturing it, without the host copies and with the bounds of every replay. */
typedef struct gla_decode_shared_args {
    gla_decode_args decode;     /* the batch, as gla_decode takes it; its windows count from the sequence's start */
    int n_groups;
    const int32_t *group_start; /* device int32[n_groups + 1], rising, within 0 .. n_seqs */
    const int32_t *prefix_len;  /* device int32[n_groups]: positions that a group's rows share */
    int max_group;              /* host: >= the rows of every group */
    int max_prefix_len;         /* host: >= every prefix_len */
    int max_own_len;            /* host: >= kv_start + kv_len - prefix_len of every row (0 for one that ends sooner;
                                   prefix_len 0 for rows in no group) */
    const int32_t *group_start_host; /* optional host copies, both or neither, */
    const int32_t *prefix_len_host;  /* beside decode's: read during the call */
} gla_decode_shared_args;

int gla_decode_shared(gla_ctx *ctx, const gla_decode_shared_args *args);

/* Host-buffer mirror of GpuBackend::attention (src/backend/gpu.rs:266-397):
 * q [n_heads][head_dim]; k, v [seq_len][n_kv_heads][head_dim]; out
 * [n_heads][head_dim]. Adds the soft-cap the wgpu shader lacks and has no
 * MAX_SEQ limit. Returns when `out` is filled. */
int gla_attention(gla_ctx *ctx, const float *q, const float *k, const float *v, int n_heads, int n_kv_heads,
                  int head_dim, int seq_len, float scale, float softcap, float *out);

/* Host-buffer mirror of GpuBackend::attention_resident
 * (src/backend/gpu.rs:860-992) over a device-resident contiguous cache:
 * attends [window_start, window_start + attend_len) of (seq, layer). */
int gla_attention_resident(gla_ctx *ctx, const float *q, const gla_kv *cache, int seq, int layer,
                           int window_start, int attend_len, int n_heads, float scale, float softcap,
                           float *out);

/* ---- the ops beside attention on a decode step --------------------------- */

/* RoPE in place, ops::rope (src/tensor/ops.rs:212-245) on device rows:
 * x [n_rows][n_heads][head_dim], row r at position pos[r] (device int32).
 * For even i < min(rot_dim, head_dim) & ~1 every head's pair (i, i+1) is
 * rotated by (pos / scaling_factor) * (1 / powf(freq_base, i / head_dim)),
 * the frequency taken from the host's powf as the reference's f32::powf
 * takes it; the other dimensions are left as they are. Like the reference,
 * freq_base and scaling_factor are not validated. Asynchronous; no device
 * allocation or copy (the frequencies travel as kernel arguments). */
int gla_rope(gla_ctx *ctx, float *x, int n_rows, int n_heads, int head_dim, const int32_t *pos, float freq_base,
             float scaling_factor, int rot_dim);

/* Rotary positions beyond gla_rope's: both layouts, part of the head, and
 * frequencies stretched for contexts longer than the model was trained on.
 * Pair p < rot_dim / 2 of a head at position pos is turned by the angle
 * pos * f[p]:
 *     (a, b) -> amplitude * (a cos - b sin, a sin + b cos),
 * (a, b) = dimensions (2p, 2p + 1) in the interleaved layout and
 * (p, p + rot_dim / 2) in the half layout; dimensions from rot_dim on are left
 * as they are. Angles, cos, sin and the products are 64-bit; the result is
 * rounded once. Positions may be negative (turning back). */
typedef enum gla_rope_layout { GLA_ROPE_INTERLEAVED = 0, GLA_ROPE_HALF = 1 } gla_rope_layout;
/* From the frequency g = freq_base^(-2p / freq_dim) / divisors[p]:
 *   NONE    f = g
 *   LINEAR  f = g / factor
 *   BANDS   by the turns t = original_ctx * g / 2 pi a pair makes in the
 *           original context: f = g / factor below `low` turns, g above
 *           `high`, between them (1 - w) g / factor + w g,
 *           w = (t - low) / (high - low)
 *   YARN    by the pair: w falls linearly from 1 at pair
 *           max(floor(e(high)), 0) to 0 at pair min(ceil(e(low)),
 *           freq_dim - 1) (0.001 pairs later where the two are equal), where
 *           e(t) is the pair that would make t turns,
 *           freq_dim * ln(original_ctx / (2 pi t)) / (2 ln freq_base);
 *           f = (1 - w) g / factor + w g; the amplitude's default is
 *           0.1 ln(factor) + 1 (for factor > 1) */
typedef enum gla_rope_scaling {
    GLA_ROPE_NONE = 0,
    GLA_ROPE_LINEAR = 1,
    GLA_ROPE_BANDS = 2,
    GLA_ROPE_YARN = 3
} gla_rope_scaling;
typedef struct gla_rope_spec {
    int head_dim; /* 1 .. 256 */
    int rot_dim;  /* rotated dimensions of a head, even, <= head_dim; 0: all (head_dim even) */
    int freq_dim; /* the exponent's denominator; 0: rot_dim (gla_rope's is head_dim) */
    gla_rope_layout layout;
    gla_rope_scaling scaling;
    int original_ctx;      /* BANDS, YARN: positions the model was trained on */
    double freq_base;      /* > 0; for YARN not 1 */
    double factor;         /* LINEAR, BANDS, YARN: > 0 */
    double low, high;      /* BANDS, YARN: turns, 0 < low < high */
    double amplitude;      /* of cos and sin; 0: the rule's own (1, for YARN see above) */
    const float *divisors; /* host [rot_dim / 2], none of them 0 (a GGUF file's rope_freqs), or NULL */
} gla_rope_spec;
/* The frequencies f[rot_dim / 2] and the amplitude a specification gives
 * (either output may be NULL). Host only: needs no device. */
int gla_rope_freqs(const gla_rope_spec *spec, double *freqs, double *amplitude);

/* A specification's frequencies on the device, made once per model. Freed
 * with its context or by gla_rope_plan_destroy, like the weights below. */
typedef struct gla_rope_plan gla_rope_plan;
int gla_rope_plan_create(gla_ctx *ctx, const gla_rope_spec *spec, gla_rope_plan **out);
int gla_rope_plan_destroy(gla_rope_plan *plan);

/* Rotate device rows: x [n_rows] rows of [n_heads][head_dim] floats, x_stride
 * floats apart (0: n_heads * head_dim), into out likewise; row r at position
 * pos[r] (device int32). out may be x with the same stride (in place); other
 * overlaps are not allowed. At most 33,554,428 rows a call (else
 * GLA_ERR_INVALID: split it). Asynchronous; allocates nothing. */
int gla_rope_rows(gla_ctx *ctx, const gla_rope_plan *plan, const float *x, int64_t x_stride, float *out,
                  int64_t out_stride, int n_rows, int n_heads, const int32_t *pos);

/* Append new positions to the caches or page tables of a batch, from the rows
 * a fused Q/K/V projection gives: K rotated on the way, V as it is, both
 * quantised for Q8_0 storage as gla_kv_write_rows does (bit for bit), and the
 * queries rotated beside them into the dense rows gla_decode and gla_prefill
 * take. Sequence b's new rows are q_start[b] .. q_start[b+1]-1 of k, v and q,
 * row r at position pos_offset[b] + (r - q_start[b]), as in gla_prefill; a
 * decode step has one row per sequence.
 * K and V of a row whose position is outside the storage (a cache's max_seq, a
 * pool's page_table_stride * 16 positions), whose seq_slot is no sequence or
 * whose page id is no page are not stored (the reference panics; a clamped
 * write would overwrite another row); its query is rotated all the same. Where
 * rows of one call meet at one place of the storage (a page in two tables), every
 * stored value is one of theirs, which one is unspecified and may differ from value
 * to value (a Q8_0 quant may lie beside another row's scale): give each sequence
 * pages of its own first. Rows past max_q_len of a sequence and rows outside every
 * sequence are left alone. Asynchronous; allocates nothing. */
typedef struct gla_append_args {
    gla_kv *kv;
    int layer;                 /* caches */
    int n_seqs;                /* B, at most 2,147,450,880 */
    const int32_t *seq_slot;   /* caches: device int32[B] or NULL */
    const int32_t *page_table; /* pools: device int32[B][page_table_stride] */
    int page_table_stride;
    const int32_t *q_start;    /* device int32[B + 1] */
    const int32_t *pos_offset; /* device int32[B] */
    int max_q_len;             /* host: >= every q_start[b+1] - q_start[b] */
    const gla_rope_plan *rope; /* NULL: no rotation; else its head_dim is the storage's */
    const float *k;            /* device rows of [n_kv_heads][head_dim], k_stride floats apart (0: dense) */
    int64_t k_stride;
    const float *v;            /* the same */
    int64_t v_stride;
    const float *q;            /* device rows of [n_heads][head_dim], q_stride floats apart (0: dense), or NULL */
    int64_t q_stride;
    float *q_out;              /* device [rows][n_heads][head_dim]; q itself where that is dense, else apart from q, k and v */
    int n_heads;               /* of q */
} gla_append_args;
int gla_kv_append(gla_ctx *ctx, const gla_append_args *args);

/* Q8_0 weights on the device, uploaded once: the GpuBackend::upload_buffer of
 * a GGML Q8_0 tensor (src/backend/gpu.rs:111-121), repacked for the MFMA
 * matvec. ggml_host: rows x (cols / 32) blocks of [f16 scale LE][32 x i8]
 * (34 bytes); cols a multiple of 32. Returns when the weights are on the
 * device. */
typedef struct gla_q8w gla_q8w;
int gla_q8w_create(gla_ctx *ctx, const uint8_t *ggml_host, int rows, int cols, gla_q8w **out);
int gla_q8w_destroy(gla_q8w *w);
int gla_q8w_rows(const gla_q8w *w);
int gla_q8w_cols(const gla_q8w *w);

/* y[v][r] = sum_c W[r][c] * x[v][c] for n_vec vectors: QuantizedTensor::matvec
 * and matvec_batch over Q8_0 (src/tensor/quantized.rs:247-346, :587-610; the
 * wgpu matvec_q8_0 shader's job). x device [n_vec][cols], y device
 * [n_vec][rows], f32. Asynchronous; up to 64 vectors read the weights
 * once, more share them in tiles through LDS. n_vec above 262,128 is refused
 * (GLA_ERR_INVALID): split the call. */
int gla_matvec_q8_0(gla_ctx *ctx, const gla_q8w *w, const float *x, int n_vec, float *y);

/* 4-bit weights on the device, uploaded once from a GGML tensor and repacked:
 *   Q4_0  rows x (cols / 32) blocks of 18 bytes, [f16 d][16 bytes: low nibbles
 *         values 0-15, high nibbles 16-31], value d * (nibble - 8)
 *   Q4_K  rows x (cols / 256) blocks of 144 bytes, [f16 d][f16 dmin][12 bytes:
 *         eight 6-bit scales and eight 6-bit minima][128 bytes of nibbles],
 *         value (d * scale) * nibble - dmin * minimum in groups of 32
 * cols a multiple of 32 (Q4_0) or 256 (Q4_K); rows and cols at most 2^26, and
 * rows * cols about 2^37 (GLA_ERR_INVALID above). Returns when the weights are on
 * the device; handles behave as gla_q8w's do. */
typedef enum gla_q4_format { GLA_Q4_0 = 0, GLA_Q4_K = 1 } gla_q4_format;
typedef struct gla_q4w gla_q4w;
int gla_q4w_create(gla_ctx *ctx, gla_q4_format format, const uint8_t *ggml_host, int rows, int cols, gla_q4w **out);
int gla_q4w_destroy(gla_q4w *w);
int gla_q4w_rows(const gla_q4w *w);
int gla_q4w_cols(const gla_q4w *w);

/* y[v][r] = sum_c W[r][c] * x[v][c] for n_vec vectors. A vector's outputs do not
 * depend on the others' values, but their rounding depends on n_vec (unlike
 * gla_matvec_q8_0's from 5 vectors on): calls of different n_vec agree to f32
 * rounding of the sum of |W[r][c] * x[v][c]| (for Q4_K of its nibbles' and its
 * minima's parts), not bit for bit. x counts with 22 bits, and with an absolute
 * error of 2^-38 of the largest |x| of its vector where that is more.
 * x device [n_vec][cols], y device [n_vec][rows], f32, y apart from x. Infinite
 * and NaN elements of x act as in that sum (infinity times a weight of 0 is NaN)
 * and stay in their vector's outputs.
 * Asynchronous; up to 8 vectors allocate nothing, more take scratch of the
 * stream, which the first call of a size allocates: make that call before
 * capturing it into a graph (a capture that would allocate is refused,
 * GLA_ERR_INVALID; partial sums that alone would not fit are done without, the
 * same bits in two launches). n_vec above 262,128 is refused (split the call). */
int gla_matvec_q4(gla_ctx *ctx, const gla_q4w *w, const float *x, int n_vec, float *y);

/* Norms around a transformer block in one pass over device rows of `dim` floats:
 *     z        = post ? y / sqrt(mean(y^2) + eps) * post : y     (the block's output, normed)
 *     x_out    = x + scale * gate * z                            (the residual stream)
 *     norm_out = x_out / sqrt(mean(x_out^2) + eps) * pre         (the next block's input)
 * the rms_norm and add shaders' job (src/backend/shaders) with what models put
 * between them. y NULL: the stream stays x (post and gate NULL too). x_out or
 * norm_out may be NULL; pre and norm_out come together. Strides are floats from row
 * to row, 0: dim; gate_stride 0: one gate for all rows. An output may be x, y or a
 * gate of rows, row for row (the same address and stride), or apart from all inputs
 * and the other output; other overlaps are refused. Sums of squares are in 32 bits;
 * a NaN or an infinity stays in its row. dim at most GLA_BLOCK_NORM_MAX_DIM;
 * 16-byte aligned rows and strides are faster. Asynchronous; allocates nothing. */
#define GLA_BLOCK_NORM_MAX_DIM 16384
typedef struct gla_block_norm_args {
    int n_rows;
    int dim;
    float eps;
    float scale;
    const float *x; /* device rows */
    int64_t x_stride;
    const float *y; /* device rows or NULL */
    int64_t y_stride;
    const float *post; /* device [dim] or NULL */
    const float *gate; /* device rows, or [dim] with gate_stride 0, or NULL */
    int64_t gate_stride;
    const float *pre; /* device [dim] or NULL */
    float *x_out;     /* device rows or NULL */
    int64_t x_out_stride;
    float *norm_out; /* device rows or NULL */
    int64_t norm_out_stride;
} gla_block_norm_args;
int gla_block_norm(gla_ctx *ctx, const gla_block_norm_args *args);

#ifdef __cplusplus
}
#endif

#endif /* GLINT_ATTN_H */
