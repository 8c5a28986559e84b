// gla_norm.hip -- norms around a transformer block, its gate and the residual sum, in
// one pass over the rows (gfx950, HBM-bound; one row: launch and latency).
//
// Math, row by row:
//   z  = post ? y / sqrt(mean(y^2) + eps) * post : y
//   x' = x + scale * gate * z
//   h  = x' / sqrt(mean(x'^2) + eps) * pre
// A row is held in registers from its loads to its stores, so the stream and the
// block's output are read once and the second norm needs no second read; both sums of
// squares are 32-bit trees over the row's threads.
#include <math.h>

#include <algorithm>

#include "gla_internal.h"

namespace gla {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

struct NormParams {
    const float *x, *y, *post, *gate, *pre;
    float *x_out, *norm_out;
    int64_t x_stride, y_stride, gate_stride, x_out_stride, norm_out_stride;
    int n_rows, dim;
    float eps, scale;
};

// Sum over the T threads of a row (whole waves); `lds` is used by rows of several waves.
template <int T>
__device__ __forceinline__ float row_sum(float v, float *lds) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if constexpr (T > 64) {
        constexpr int W = T / 64;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < W; w++) v += lds[w];
    }
    return v;
}

// T threads a row, N pieces of E floats (1 or 4) a thread.
template <int T, int N, int E>
__global__ __launch_bounds__(T < 256 ? 256 : T) void block_norm_kernel(const NormParams p) {
    typedef float vec __attribute__((ext_vector_type(E == 4 ? 4 : 2)));  // (E == 1 goes by single floats)
    constexpr int RPW = T < 256 ? 256 / T : 1;  // rows per workgroup
    __shared__ float lds[2][T / 64];
    const int t = threadIdx.x % T;
    const int pieces = p.dim / E;
    const auto load = [&](const float *row, int k, float (&v)[E]) {
        const int i = t + k * T;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = 0.0f;
        if (i < pieces) {
            if constexpr (E == 4) {
                const vec w = *reinterpret_cast<const vec *>(row + 4 * i);
#pragma unroll
                for (int e = 0; e < E; e++) v[e] = w[e];
            } else {
                v[0] = row[i];
            }
        }
    };
    const auto store = [&](float *row, int k, const float (&v)[E]) {
        const int i = t + k * T;
        if (i < pieces) {
            if constexpr (E == 4)
                *reinterpret_cast<vec *>(row + 4 * i) = vec{v[0], v[1], v[2], v[3]};
            else
                row[i] = v[0];
        }
    };
    const auto squares = [&](const float (&v)[N][E]) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < E; e++) s = fmaf(v[k][e], v[k][e], s);
        return s;
    };
    for (int64_t r = (int64_t)blockIdx.x * RPW + threadIdx.x / T; r < p.n_rows; r += (int64_t)gridDim.x * RPW) {
        float x[N][E], y[N][E];
#pragma unroll
        for (int k = 0; k < N; k++) load(p.x + r * p.x_stride, k, x[k]);
        if (p.y) {
#pragma unroll
            for (int k = 0; k < N; k++) load(p.y + r * p.y_stride, k, y[k]);
            if (p.gate) {
                float g[N][E];
#pragma unroll
                for (int k = 0; k < N; k++) load(p.gate + r * p.gate_stride, k, g[k]);
                float f = p.scale;
                if (p.post) f *= 1.0f / sqrtf(row_sum<T>(squares(y), lds[0]) / (float)p.dim + p.eps);
#pragma unroll
                for (int k = 0; k < N; k++)
#pragma unroll
                    for (int e = 0; e < E; e++) y[k][e] *= g[k][e] * f;
            } else {
                float f = p.scale;
                if (p.post) f *= 1.0f / sqrtf(row_sum<T>(squares(y), lds[0]) / (float)p.dim + p.eps);
#pragma unroll
                for (int k = 0; k < N; k++)
#pragma unroll
                    for (int e = 0; e < E; e++) y[k][e] *= f;
            }
            if (p.post) {
#pragma unroll
                for (int k = 0; k < N; k++) {
                    float w[E];
                    load(p.post, k, w);
#pragma unroll
                    for (int e = 0; e < E; e++) x[k][e] = fmaf(y[k][e], w[e], x[k][e]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < N; k++)
#pragma unroll
                    for (int e = 0; e < E; e++) x[k][e] += y[k][e];
            }
        }
        if (p.x_out) {
#pragma unroll
            for (int k = 0; k < N; k++) store(p.x_out + r * p.x_out_stride, k, x[k]);
        }
        if (p.norm_out) {
            const float f = 1.0f / sqrtf(row_sum<T>(squares(x), lds[1]) / (float)p.dim + p.eps);
#pragma unroll
            for (int k = 0; k < N; k++) {
                float w[E];
                load(p.pre, k, w);
#pragma unroll
                for (int e = 0; e < E; e++) x[k][e] *= f * w[e];
                store(p.norm_out + r * p.norm_out_stride, k, x[k]);
            }
        }
        if constexpr (T > 64) __syncthreads();  // the sums are read: the next row may write them
    }
}

template <int T, int N, int E>
int launch_as(gla_ctx *ctx, const NormParams &p) {
    constexpr int RPW = T < 256 ? 256 / T : 1;
    const int64_t wgs = ((int64_t)p.n_rows + RPW - 1) / RPW;
    hipLaunchKernelGGL((block_norm_kernel<T, N, E>), dim3((unsigned)std::min<int64_t>(wgs, 1 << 20)),
                       dim3(T < 256 ? 256 : T), 0, ctx->stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(GLA_ERR_KERNEL, "block_norm_kernel launch: %s", hipGetErrorString(e));
    return GLA_OK;
}

template <int E>
int launch_e(gla_ctx *ctx, const NormParams &p) {
    const int pieces = p.dim / E;
    if (pieces <= 64) return launch_as<64, 1, E>(ctx, p);
    if (pieces <= 256) return launch_as<64, 4, E>(ctx, p);
    if (pieces <= 1024) return launch_as<256, 4, E>(ctx, p);
    if (pieces <= 4096) return launch_as<1024, 4, E>(ctx, p);
    if constexpr (E == 1) return launch_as<1024, 16, 1>(ctx, p);
    return set_error(GLA_ERR_INVALID, "gla_block_norm: dim %d", p.dim);
}

// Device rows of an argument, `stride` floats apart.
struct Rows {
    const float *at;
    int64_t stride;
    int64_t n;
    bool same(const Rows &o) const { return at == o.at && n == o.n && (stride == o.stride || n == 1); }
    // whether a float is in rows of both (dim floats long)
    bool meets(const Rows &o, int dim) const {
        if (!at || !o.at) return false;
        const uintptr_t a = (uintptr_t)at, b = (uintptr_t)o.at;
        if (a + 4 * ((uint64_t)stride * (n - 1) + dim) <= b || b + 4 * ((uint64_t)o.stride * (o.n - 1) + dim) <= a)
            return false;
        if (stride != o.stride || n != o.n) return true;
        // columns of one wider row: none in both
        const uint64_t off = (a > b ? a - b : b - a) % (4 * (uint64_t)stride);
        return off < 4 * (uint64_t)dim || 4 * (uint64_t)stride - off < 4 * (uint64_t)dim;
    }
};

}  // namespace

}  // namespace gla

using namespace gla;

extern "C" {

int gla_block_norm(gla_ctx *ctx, const gla_block_norm_args *a) {
    GLA_GUARD_BEGIN
    GLA_REQUIRE(ctx && a, "gla_block_norm: NULL argument");
    GLA_REQUIRE(a->n_rows >= 0, "gla_block_norm: n_rows < 0");
    GLA_REQUIRE(a->dim >= 1 && a->dim <= GLA_BLOCK_NORM_MAX_DIM, "gla_block_norm: dim %d is not in 1 .. %d", a->dim,
                GLA_BLOCK_NORM_MAX_DIM);
    GLA_REQUIRE(a->eps >= 0.0f && a->eps < INFINITY, "gla_block_norm: eps must be finite and not negative");
    GLA_REQUIRE(a->y || (!a->post && !a->gate), "gla_block_norm: post and gate are of y, which is NULL");
    GLA_REQUIRE(a->x_out || a->norm_out, "gla_block_norm: no output");
    GLA_REQUIRE((a->pre != nullptr) == (a->norm_out != nullptr), "gla_block_norm: pass both pre and norm_out, or neither");
    if (a->n_rows == 0) return GLA_OK;
    GLA_REQUIRE(a->x, "gla_block_norm: NULL buffer");
    NormParams p;
    p.x = a->x;
    p.y = a->y;
    p.post = a->post;
    p.gate = a->gate;
    p.pre = a->pre;
    p.x_out = a->x_out;
    p.norm_out = a->norm_out;
    p.x_stride = a->x_stride ? a->x_stride : a->dim;
    p.y_stride = a->y_stride ? a->y_stride : a->dim;
    p.gate_stride = a->gate_stride;
    p.x_out_stride = a->x_out_stride ? a->x_out_stride : a->dim;
    p.norm_out_stride = a->norm_out_stride ? a->norm_out_stride : a->dim;
    const int64_t least = a->dim;
    GLA_REQUIRE(p.x_stride >= least && p.x_out_stride >= least && p.norm_out_stride >= least && p.y_stride >= least &&
                    (p.gate_stride == 0 || p.gate_stride >= least),
                "gla_block_norm: a row stride is below dim %d", a->dim);
    // A row is read before it is written: an output may take an input's place, row for row.
    const Rows x_out = {a->x_out, p.x_out_stride, a->n_rows}, norm_out = {a->norm_out, p.norm_out_stride, a->n_rows};
    const Rows ins[] = {{a->x, p.x_stride, a->n_rows},
                        {a->y, p.y_stride, a->n_rows},
                        {a->gate, p.gate_stride, p.gate_stride ? a->n_rows : 1}};
    for (const Rows &in : ins)
        for (const Rows &out : {x_out, norm_out})
            GLA_REQUIRE(out.same(in) || !out.meets(in, a->dim),
                        "gla_block_norm: an output overlaps an input other than row for row");
    const Rows post = {a->post, least, 1}, pre = {a->pre, least, 1};
    for (const Rows &out : {x_out, norm_out})
        GLA_REQUIRE(!out.meets(post, a->dim) && !out.meets(pre, a->dim), "gla_block_norm: an output overlaps a weight");
    GLA_REQUIRE(!x_out.meets(norm_out, a->dim), "gla_block_norm: x_out and norm_out overlap");
    p.n_rows = a->n_rows;
    p.dim = a->dim;
    p.eps = a->eps;
    p.scale = a->scale;
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    const auto aligned = [](const float *q, int64_t stride) { return ((uintptr_t)q & 15) == 0 && stride % 4 == 0; };
    const bool four = a->dim % 4 == 0 && aligned(p.x, p.x_stride) && (!p.y || aligned(p.y, p.y_stride)) &&
                      aligned(p.post, 0) && aligned(p.gate, p.gate_stride) && aligned(p.pre, 0) &&
                      (!p.x_out || aligned(p.x_out, p.x_out_stride)) &&
                      (!p.norm_out || aligned(p.norm_out, p.norm_out_stride));
    return four ? launch_e<4>(ctx, p) : launch_e<1>(ctx, p);
    GLA_GUARD_END
}

}  // extern "C"
