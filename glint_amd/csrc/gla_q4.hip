// gla_q4.hip -- projections with 4-bit weights: GGML's Q4_0 (groups of 32 with
// an f16 scale) and Q4_K (groups of 32 with a 6-bit scale and minimum, eight of
// them under an f16 scale of each kind).
//
// Weights are repacked once, on upload, into pieces of 16 rows x 128 columns (a
// row tile and a quad of groups), in the operand order of
// v_mfma_f32_16x16x32_f16: lane l of a wave holds row l % 16, and of each of the
// four groups elements (l / 16) * 8 .. +8 as one dword, so a wave reads a piece
// as one contiguous kilobyte. Element 2i of the eight sits at bits 4i of its
// dword and element 2i + 1 at bits 16 + 4i: two masks give both as halves.
//   quants [tile][quad][64 lanes][4 groups] u32
//   aux    [tile][quad][16 rows] 8 bytes: Q4_0 four f16 scales; Q4_K four scale
//          bytes, then four minimum bytes
//   super  Q4_K: [tile][superblock][16 rows] {f16 d, f16 dmin}
// Groups and rows past the matrix have scale (and minimum) 0.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "gla_internal.h"

struct gla_q4w {
    gla_ctx *ctx = nullptr;
    gla_q4_format format = GLA_Q4_0;
    int rows = 0;
    int cols = 0;
    int n_tiles = 0;  // ceil(rows / 16)
    int n_quads = 0;  // ceil(cols / 128)
    uint8_t *quants = nullptr;
    uint8_t *aux = nullptr;
    uint32_t *super = nullptr;
};

namespace gla {

void detach_q4w(gla_q4w *w) {
    if (w->quants) (void)hipFree(w->quants);
    if (w->aux) (void)hipFree(w->aux);
    if (w->super) (void)hipFree(w->super);
    w->quants = w->aux = nullptr;
    w->super = nullptr;
    w->ctx = nullptr;
}

namespace {

struct Weights {
    const uint8_t *quants;
    const uint8_t *aux;
    const uint32_t *super;
    int rows, cols, n_tiles, n_quads;
};

// ---- repack ----------------------------------------------------------------------

// One thread per (tile, quad, lane): the lane's four dwords and, of lanes 0..15,
// the 8 aux bytes of row tile * 16 + lane and the superblock's word.
template <bool K>
__global__ __launch_bounds__(256) void q4_repack_kernel(const uint8_t *ggml, int rows, int n_groups, int n_quads,
                                                        int64_t n_units, uint8_t *quants, uint8_t *aux,
                                                        uint32_t *super) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= n_units) return;
    const int lane = (int)(u & 63);
    const int64_t tq = u >> 6;
    const int quad = (int)(tq % n_quads);
    const int tile = (int)(tq / n_quads);
    const int row = tile * 16 + (lane & 15);
    const int k8 = (lane >> 4) * 8;  // first of the lane's elements in a group
    uint32_t w[4];
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int g = quad * 4 + j;
        w[j] = 0;
        if (row >= rows || g >= n_groups) continue;
        const uint8_t *blk;  // the group's nibbles: 16 bytes low then high (Q4_0), 32 bytes low or high (Q4_K)
        if (K)
            blk = ggml + ((int64_t)row * (n_groups / 8) + g / 8) * 144;
        else
            blk = ggml + ((int64_t)row * n_groups + g) * 18;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int k = k8 + e;
            uint32_t q;
            if (K)
                q = (blk[16 + (g % 8 / 2) * 32 + k] >> (g % 2 * 4)) & 15u;
            else
                q = (blk[2 + k % 16] >> (k / 16 * 4)) & 15u;
            w[j] |= q << (e / 2 * 4 + e % 2 * 16);
        }
        if (K) {
            const uint8_t *b = blk + 4;
            const int i = g % 8;
            const uint32_t sc = i < 4 ? b[i] & 63u : (b[i + 4] & 15u) | (uint32_t)(b[i - 4] >> 6) << 4;
            const uint32_t mn = i < 4 ? b[i + 4] & 63u : (uint32_t)(b[i + 4] >> 4) | (uint32_t)(b[i] >> 6) << 4;
            lo |= sc << (8 * j);
            hi |= mn << (8 * j);
            if (lane < 16 && g % 8 == 0)
                super[((int64_t)tile * (n_quads / 2) + g / 8) * 16 + lane] =
                    blk[0] | (uint32_t)blk[1] << 8 | (uint32_t)blk[2] << 16 | (uint32_t)blk[3] << 24;
        } else {
            const uint32_t d = blk[0] | (uint32_t)blk[1] << 8;
            (j < 2 ? lo : hi) |= d << (j % 2 * 16);
        }
    }
    *reinterpret_cast<uint4 *>(quants + u * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    if (lane < 16) {
        *reinterpret_cast<uint2 *>(aux + (tq * 16 + lane) * 8) = make_uint2(lo, hi);
        if (K && row >= rows && quad % 2 == 0) super[((int64_t)tile * (n_quads / 2) + quad / 2) * 16 + lane] = 0;
    }
}

// ---- the product --------------------------------------------------------------------

__device__ __forceinline__ float half_of(uint32_t w, int hi) {
    return __half2float(__ushort_as_half((unsigned short)(hi ? w >> 16 : w & 0xffffu)));
}

// y[v][row], one wave per row tile, up to 4 vectors a workgroup row: each lane
// multiplies its row's elements in f32 and the four element groups are summed.
template <bool K>
__global__ __launch_bounds__(64) void matvec_q4_plain_kernel(const Weights w, const float *x, int n_vec, float *y) {
    const int lane = threadIdx.x;
    const int tile = blockIdx.x;
    const int r = lane & 15, kg = lane >> 4;
    const int v0 = blockIdx.y * 4;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int quad = 0; quad < w.n_quads; quad++) {
        const int64_t tq = (int64_t)tile * w.n_quads + quad;
        const uint4 q = *reinterpret_cast<const uint4 *>(w.quants + (tq * 64 + lane) * 16);
        const uint2 a = *reinterpret_cast<const uint2 *>(w.aux + (tq * 16 + r) * 8);
        const uint32_t sup = K ? w.super[((int64_t)tile * (w.n_quads / 2) + quad / 2) * 16 + r] : 0;
        const uint32_t qs[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = quad * 128 + j * 32 + kg * 8;
            if (c >= w.cols) continue;
            const float s = K ? half_of(sup, 0) * (float)((a.x >> (8 * j)) & 255u) : half_of(j < 2 ? a.x : a.y, j & 1);
            const float m = K ? half_of(sup, 1) * (float)((a.y >> (8 * j)) & 255u) : 0.0f;
#pragma unroll
            for (int v = 0; v < 4; v++) {
                if (v0 + v >= n_vec) continue;
                const float *xv = x + (int64_t)(v0 + v) * w.cols + c;
                float t = 0.0f, sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float n = (float)((qs[j] >> (e / 2 * 4 + e % 2 * 16)) & 15u) - (K ? 0.0f : 8.0f);
                    t = fmaf(n, xv[e], t);
                    sum += xv[e];
                }
                acc[v] = fmaf(t, s, acc[v]);
                if (K) acc[v] = fmaf(-sum, m, acc[v]);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < 4; v++) {
        acc[v] += __shfl_xor(acc[v], 16);
        acc[v] += __shfl_xor(acc[v], 32);
        const int row = tile * 16 + r;
        if (kg == 0 && row < w.rows && v0 + v < n_vec) y[(int64_t)(v0 + v) * w.rows + row] = acc[v];
    }
}

constexpr int kMaxVec = 262128;

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GLA_OK : set_error(GLA_ERR_KERNEL, "%s launch: %s", what, hipGetErrorString(e));
}

}  // namespace
}  // namespace gla

using namespace gla;

extern "C" {

int gla_q4w_create(gla_ctx *ctx, gla_q4_format format, const uint8_t *ggml_host, int rows, int cols, gla_q4w **out) {
    GLA_GUARD_BEGIN
    GLA_REQUIRE(ctx && ggml_host && out, "gla_q4w_create: NULL argument");
    *out = nullptr;
    GLA_REQUIRE(format == GLA_Q4_0 || format == GLA_Q4_K, "gla_q4w_create: bad format %d", (int)format);
    const bool k = format == GLA_Q4_K;
    GLA_REQUIRE(rows > 0 && cols > 0 && cols % (k ? 256 : 32) == 0,
                "gla_q4w_create: rows %d, cols %d (cols must be a positive multiple of %d)", rows, cols, k ? 256 : 32);
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    ctx->q4ws.reserve(ctx->q4ws.size() + 1);
    gla_q4w *w = new gla_q4w();
    w->ctx = ctx;
    w->format = format;
    w->rows = rows;
    w->cols = cols;
    w->n_tiles = (rows + 15) / 16;
    w->n_quads = (cols + 127) / 128;
    const int n_groups = cols / 32;
    const int64_t pieces = (int64_t)w->n_tiles * w->n_quads;
    const size_t raw_bytes = (size_t)rows * (k ? (size_t)(cols / 256) * 144 : (size_t)n_groups * 18);
    uint8_t *raw = nullptr;
    hipError_t e = hipMalloc(&w->quants, (size_t)pieces * 1024);
    if (e == hipSuccess) e = hipMalloc(&w->aux, (size_t)pieces * 128);
    if (e == hipSuccess && k) e = hipMalloc(&w->super, (size_t)pieces / 2 * 64);
    if (e == hipSuccess) e = hipMalloc(&raw, raw_bytes);
    if (e == hipSuccess) e = hipMemcpyAsync(raw, ggml_host, raw_bytes, hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) {
        const int64_t n_units = pieces * 64;
        auto kernel = k ? q4_repack_kernel<true> : q4_repack_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((n_units + 255) / 256)), dim3(256), 0, ctx->stream, raw, rows, n_groups,
                           w->n_quads, n_units, w->quants, w->aux, w->super);
        e = hipGetLastError();
    }
    const hipError_t done = hipStreamSynchronize(ctx->stream);
    if (e == hipSuccess) e = done;
    if (raw) (void)hipFree(raw);
    if (e != hipSuccess) {
        (void)hipGetLastError();  // not the next launch's
        detach_q4w(w);
        delete w;
        return set_error(GLA_ERR_BUFFER, "gla_q4w_create: %s", hipGetErrorString(e));
    }
    ctx->q4ws.push_back(w);
    *out = w;
    return GLA_OK;
    GLA_GUARD_END
}

int gla_q4w_destroy(gla_q4w *w) {
    GLA_GUARD_BEGIN
    if (!w) return GLA_OK;
    if (gla_ctx *ctx = w->ctx) {  // else its context already freed the weights
        (void)hipSetDevice(ctx->device);
        (void)hipStreamSynchronize(ctx->stream);
        ctx->q4ws.erase(std::remove(ctx->q4ws.begin(), ctx->q4ws.end(), w), ctx->q4ws.end());
        detach_q4w(w);
    }
    delete w;
    return GLA_OK;
    GLA_GUARD_END
}

int gla_q4w_rows(const gla_q4w *w) { return w ? w->rows : -1; }
int gla_q4w_cols(const gla_q4w *w) { return w ? w->cols : -1; }

int gla_matvec_q4(gla_ctx *ctx, const gla_q4w *w, const float *x, int n_vec, float *y) {
    GLA_GUARD_BEGIN
    GLA_REQUIRE(ctx && w, "gla_matvec_q4: NULL argument");
    GLA_REQUIRE(w->ctx == ctx, "gla_matvec_q4: the weights belong to %s",
                w->ctx ? "another context" : "a destroyed context");
    GLA_REQUIRE(n_vec >= 0 && n_vec <= kMaxVec, "gla_matvec_q4: n_vec %d (0 to %d; split the call)", n_vec, kMaxVec);
    if (n_vec == 0) return GLA_OK;
    GLA_REQUIRE(x && y, "gla_matvec_q4: NULL buffer");
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    const Weights p{w->quants, w->aux, w->super, w->rows, w->cols, w->n_tiles, w->n_quads};
    for (int v0 = 0; v0 < n_vec; v0 += 4 * 65535) {
        const int n = std::min(n_vec - v0, 4 * 65535);
        auto kernel = w->format == GLA_Q4_K ? matvec_q4_plain_kernel<true> : matvec_q4_plain_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3(w->n_tiles, (n + 3) / 4), dim3(64), 0, ctx->stream, p, x + (int64_t)v0 * w->cols, n,
                           y + (int64_t)v0 * w->rows);
    }
    return launched("matvec_q4_plain_kernel");
    GLA_GUARD_END
}

}  // extern "C"
