// gla_kvstore.hip -- device side of KvStore::write / export_raw / import_raw,
// of reading rows back as f32 and of the page pool's copy-on-write and recycle
// wipe. Quantize-on-write (gla_rows.h) is KvCacheQ8::quantize_into's, bit for bit.
#include <algorithm>

#include "gla_rows.h"

namespace gla {

namespace {

// One thread per 8 elements of a row's K or V, so a wave reads 2 KiB of a source
// row at once and a Q8_0 block is four neighbouring lanes, which find its
// maximum with two DPP exchanges. A workgroup takes `per` whole rows (one where
// a row has 256 threads' work or more). The source does not depend on the row
// id, so both loads share one round trip. Bound: launch and latency for a
// decode step's few rows, memory for a prompt's (the V bytes of Q8_0 go out one
// by one). us per call at 8 heads x 128, against one thread per 32-element
// block: f32 4 rows 4.8 -> 3.9, 16,384 rows 220 -> 41 (6.6 TB/s); Q8_0 4 rows
// 6.7 -> 3.7, 16,384 rows 68 -> 52, 65,536 rows 349 -> 274 (2.5 TB/s).
__global__ __launch_bounds__(256) void write_rows_kernel(const RowOps o, const int64_t *rows, const float *k,
                                                         const float *v, int n, int per) {
    const int units = o.kv_dim / 4;  // 8-element units of K, then of V
    const int first = blockIdx.x * per;
    for (int t = threadIdx.x; t < units * per; t += 256) {
        const int rr = t / units;
        const int r = first + rr;
        const int u = t - rr * units;
        const int which = u >= units / 2;
        const int gi = (which ? u - units / 2 : u) * 8;
        // a block's four lanes run together: units is a multiple of 4
        if (r >= n) continue;
        const int64_t row = rows[r];
        const float4 *src = reinterpret_cast<const float4 *>((which ? v : k) + (int64_t)r * o.kv_dim + gi);
        const float4 a = src[0], c = src[1];
        if (row < 0 || row >= o.n_rows_total) continue;
        uint8_t *dst = const_cast<uint8_t *>(which ? o.L.v : o.L.k);
        if (!o.q8) {
            float4 *d = reinterpret_cast<float4 *>(dst + elem_off(o, row, gi, 4));
            d[0] = a;
            d[1] = c;
            continue;
        }
        const float e[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
        store_q8(o, row, gi, which, e);
    }
}

// The f32 values of a row's K and V: one thread per 8 elements of R rows, `per`
// rows apart, so that their ids come in one round trip and their elements in the
// next. Long calls take four rows (6,144 rows of 8 x 128: Q8_0 21.0 -> 14.8 us,
// f32 20.9 -> 19.8), short ones one (64 rows 4.2 -> 3.7). A Q8_0 value is quant times f16 scale,
// exact in f32 but for its last rounding.
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float f16_of(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }
// stored byte i of w (x + 128) as x
__device__ __forceinline__ float q8_of(uint32_t w, int i) { return (float)(int8_t)((w >> (8 * i)) ^ 0x80u); }

template <bool Q8, int R>
__global__ __launch_bounds__(256) void read_rows_kernel(const RowOps o, const int64_t *rows, float *k, float *v, int n,
                                                        int per) {
    const int units = o.kv_dim / 4;
    const int first = blockIdx.x * per * R;
    for (int t = threadIdx.x; t < units * per; t += 256) {
        const int rr = t / units;
        const int u = t - rr * units;
        int64_t row[R];
        bool ok[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int r = first + i * per + rr;
            row[i] = rows[min(r, n - 1)];
            ok[i] = r < n && row[i] >= 0 && row[i] < o.n_rows_total;
            if (!ok[i]) row[i] = 0;
        }
        const int64_t at = (int64_t)(first + rr) * o.kv_dim;
        const int64_t apart = (int64_t)per * o.kv_dim;  // floats between the thread's rows
        if constexpr (!Q8) {
            // four of K and four of V
            floatx4 a[R], b[R];
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int64_t off = elem_off(o, row[i], u * 4, 4);
                a[i] = *reinterpret_cast<const floatx4 *>(o.L.k + off);
                b[i] = *reinterpret_cast<const floatx4 *>(o.L.v + off);
            }
#pragma unroll
            for (int i = 0; i < R; i++)
                if (ok[i]) {
                    *reinterpret_cast<floatx4 *>(k + at + i * apart + u * 4) = a[i];
                    *reinterpret_cast<floatx4 *>(v + at + i * apart + u * 4) = b[i];
                }
        } else if (u < units / 2) {
            const int gi = u * 8;
            u32x2 q[R];
            uint16_t sc[R];
#pragma unroll
            for (int i = 0; i < R; i++) {
                q[i] = *reinterpret_cast<const u32x2 *>(o.L.k + q8_off(o, row[i], gi, 0));
                sc[i] = *reinterpret_cast<const uint16_t *>(o.L.ks + scale_off(o, row[i], gi, 0));
            }
#pragma unroll
            for (int i = 0; i < R; i++)
                if (ok[i]) {
                    const float d = f16_of(sc[i]);
                    float *to = k + at + i * apart + gi;
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        reinterpret_cast<floatx4 *>(to)[j] =
                            floatx4{q8_of(q[i][j], 0), q8_of(q[i][j], 1), q8_of(q[i][j], 2), q8_of(q[i][j], 3)} * d;
                }
        } else {
            // a column of the page's V holds dimensions j, j + 16, j + 32, j + 48 of
            // four positions in 16 bytes: the thread takes two columns of each row
            u32x4 q[R][2];
            uint32_t sc[R][2];
            int g[2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int col = u - units / 2 + c * (units / 2);  // 16 to 64 dimensions
                g[c] = (col >> 4) * 64 + (col & 15);
#pragma unroll
                for (int i = 0; i < R; i++) {
                    q[i][c] = *reinterpret_cast<const u32x4 *>(o.L.v + (q8_off(o, row[i], g[c], 1) & ~(int64_t)15));
                    sc[i][c] = *reinterpret_cast<const uint32_t *>(o.L.vs + scale_off(o, row[i], g[c], 1));
                }
            }
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int i = 0; i < R; i++)
                    if (ok[i]) {
                        float *to = v + at + i * apart + g[c];
                        const int byte = (int)(row[i] & 3);
#pragma unroll
                        for (int m = 0; m < 4; m++)
                            to[16 * m] = q8_of(q[i][c][m], byte) * f16_of(m < 2 ? sc[i][c] : sc[i][c] >> 16);
                    }
        }
    }
}

// Export to Glint's row bytes (f32 rows, or Q8_0 34-byte blocks).
__global__ __launch_bounds__(64) void export_rows_kernel(const RowOps o, const int64_t *rows, int n,
                                                         uint8_t *k_out, uint8_t *v_out) {
    const int r = blockIdx.x;
    if (r >= n) return;
    const int64_t row = rows[r];
    if (row < 0 || row >= o.n_rows_total) return;
    const int64_t row_bytes = o.q8 ? (int64_t)o.n_blocks * 34 : (int64_t)o.kv_dim * 4;
    for (int t = threadIdx.x; t < 2 * o.n_blocks; t += blockDim.x) {
        const int which = t >= o.n_blocks;
        const int blk = which ? t - o.n_blocks : t;
        const uint8_t *src = which ? o.L.v : o.L.k;
        uint8_t *out = (which ? v_out : k_out) + (int64_t)r * row_bytes;
        const int gi0 = blk * 32;
        if (!o.q8) {
            const uint8_t *s = src + elem_off(o, row, gi0, 4);
            for (int j = 0; j < 128; j++) out[(int64_t)gi0 * 4 + j] = s[j];
        } else {
            const uint8_t *sc = (which ? o.L.vs : o.L.ks) + scale_off(o, row, gi0, which);
            uint8_t *ob = out + (int64_t)blk * 34;
            ob[0] = sc[0];
            ob[1] = sc[1];
            for (int j = 0; j < 32; j++) ob[2 + j] = src[q8_off(o, row, gi0 + j, which)] ^ 0x80;
        }
    }
}

__global__ __launch_bounds__(64) void import_rows_kernel(const RowOps o, const int64_t *rows, int n,
                                                         const uint8_t *k_in, const uint8_t *v_in) {
    const int r = blockIdx.x;
    if (r >= n) return;
    const int64_t row = rows[r];
    if (row < 0 || row >= o.n_rows_total) return;
    const int64_t row_bytes = o.q8 ? (int64_t)o.n_blocks * 34 : (int64_t)o.kv_dim * 4;
    for (int t = threadIdx.x; t < 2 * o.n_blocks; t += blockDim.x) {
        const int which = t >= o.n_blocks;
        const int blk = which ? t - o.n_blocks : t;
        uint8_t *dst = const_cast<uint8_t *>(which ? o.L.v : o.L.k);
        const uint8_t *in = (which ? v_in : k_in) + (int64_t)r * row_bytes;
        const int gi0 = blk * 32;
        if (!o.q8) {
            uint8_t *d = dst + elem_off(o, row, gi0, 4);
            for (int j = 0; j < 128; j++) d[j] = in[(int64_t)gi0 * 4 + j];
        } else {
            uint8_t *sc = const_cast<uint8_t *>(which ? o.L.vs : o.L.ks) + scale_off(o, row, gi0, which);
            const uint8_t *ib = in + (int64_t)blk * 34;
            sc[0] = ib[0];
            sc[1] = ib[1];
            for (int j = 0; j < 32; j++) dst[q8_off(o, row, gi0 + j, which)] = ib[2 + j] ^ 0x80;
        }
    }
}

// Page-granular copy and fill with 16-byte vectors (no hipMemsetAsync, so the
// calls stay valid inside a captured graph).
__global__ __launch_bounds__(256) void copy_bytes_kernel(const uint4 *src, uint4 *dst, int64_t n16) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n16; i += (int64_t)gridDim.x * blockDim.x)
        dst[i] = src[i];
}

// Fill of whole pages: a 16-byte unit at byte offset o of its (page, head)
// block of `head16` units gets `quant` below unit `quant16`, zero above (f32
// pages: everything zero; Q8_0 pages: quants 0x80 = stored 0, scales 0).
__global__ __launch_bounds__(256) void zero_bytes_kernel(uint4 *dst, int64_t n16, int64_t head16, int64_t quant16,
                                                         uint32_t quant) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n16; i += (int64_t)gridDim.x * blockDim.x) {
        const uint32_t w = (i % head16) < quant16 ? quant : 0u;
        dst[i] = make_uint4(w, w, w, w);
    }
}

int check_launch(const char *what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(GLA_ERR_KERNEL, "%s launch: %s", what, hipGetErrorString(e));
    return GLA_OK;
}

unsigned grid_for(int64_t n16) {
    int64_t blocks = (n16 + 255) / 256;
    if (blocks > 65536) blocks = 65536;
    if (blocks < 1) blocks = 1;
    return (unsigned)blocks;
}

}  // namespace

int launch_write_rows(gla_ctx *ctx, gla_kv *kv, const int64_t *rows, const float *k, const float *v, int n) {
    if (n <= 0) return GLA_OK;
    const RowOps o = row_ops(kv);
    const int per = std::max(1, 256 / (o.kv_dim / 4));
    hipLaunchKernelGGL(write_rows_kernel, dim3((n - 1) / per + 1), dim3(256), 0, ctx->stream, o, rows, k, v, n, per);
    return check_launch("write_rows_kernel");
}

int launch_read_rows(gla_ctx *ctx, const gla_kv *kv, const int64_t *rows, float *k, float *v, int n) {
    if (n <= 0) return GLA_OK;
    const RowOps o = row_ops(kv);
    const int per = std::max(1, 256 / (o.kv_dim / 4));
    const int blocks = (n - 1) / per + 1;  // of one row a thread
    const bool many = blocks >= 4 * ctx->n_cu;
    auto kernel = o.q8 ? (many ? read_rows_kernel<true, 4> : read_rows_kernel<true, 1>)
                       : (many ? read_rows_kernel<false, 4> : read_rows_kernel<false, 1>);
    hipLaunchKernelGGL(kernel, dim3(many ? (blocks + 3) / 4 : blocks), dim3(256), 0, ctx->stream, o, rows, k, v, n, per);
    return check_launch("read_rows_kernel");
}

int launch_export_rows(gla_ctx *ctx, const gla_kv *kv, const int64_t *rows, int n, uint8_t *k_out,
                       uint8_t *v_out) {
    if (n <= 0) return GLA_OK;
    const RowOps o = row_ops(kv);
    hipLaunchKernelGGL(export_rows_kernel, dim3(n), dim3(64), 0, ctx->stream, o, rows, n, k_out, v_out);
    return check_launch("export_rows_kernel");
}

int launch_import_rows(gla_ctx *ctx, gla_kv *kv, const int64_t *rows, int n, const uint8_t *k_in,
                       const uint8_t *v_in) {
    if (n <= 0) return GLA_OK;
    const RowOps o = row_ops(kv);
    hipLaunchKernelGGL(import_rows_kernel, dim3(n), dim3(64), 0, ctx->stream, o, rows, n, k_in, v_in);
    return check_launch("import_rows_kernel");
}

int launch_copy_page(gla_ctx *ctx, gla_kv *kv, int64_t src, int64_t dst) {
    const int64_t n16 = kv->page_bytes / 16;
    const uint4 *s = reinterpret_cast<const uint4 *>(kv->base + src * kv->page_bytes);
    uint4 *d = reinterpret_cast<uint4 *>(kv->base + dst * kv->page_bytes);
    hipLaunchKernelGGL(copy_bytes_kernel, dim3(grid_for(n16)), dim3(256), 0, ctx->stream, s, d, n16);
    return check_launch("copy_bytes_kernel");
}

int launch_zero_pages(gla_ctx *ctx, gla_kv *kv, int64_t first, int64_t count) {
    const int64_t n16 = kv->page_bytes / 16 * count;
    const int64_t head16 = kv->head_bytes / 16;
    const bool q8 = kv->dtype == GLA_KV_Q8_0;
    const int64_t quant16 = q8 ? (int64_t)GLA_PAGE_SIZE * kv->head_dim * 2 / 16 : 0;  // Kq and Vq
    uint4 *d = reinterpret_cast<uint4 *>(kv->base + first * kv->page_bytes);
    hipLaunchKernelGGL(zero_bytes_kernel, dim3(grid_for(n16)), dim3(256), 0, ctx->stream, d, n16, head16, quant16,
                       0x80808080u);
    return check_launch("zero_bytes_kernel");
}

}  // namespace gla
