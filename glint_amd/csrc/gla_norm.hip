// gla_norm.hip -- norms around a transformer block, its gate and the residual sum, in
// one pass over the rows (gfx950). Many rows are bound by HBM: 7,993 rows of 4,096 with
// everything, 655 MB, 104 us, 6.3 TB/s (a large copy reaches 5.1). One row is bound by its
// launch: 2.6 us in a captured step, as an empty kernel's.
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
#include "gla_lanes.h"

namespace gla {

namespace {

using namespace lanes;

typedef float floatx4 __attribute__((ext_vector_type(4)));

struct NormParams {
    const float *x, *y, *post, *gate, *pre;
    float *x_out, *norm_out;
    int64_t x_stride, y_stride, gate_stride, x_out_stride, norm_out_stride;
    int n_rows, dim;
    float eps, scale;
};

// Sum over the T threads of a row (whole waves), in every one of them; `lds` is used by
// rows of several waves.
template <int T>
__device__ __forceinline__ float row_sum(float v, float *lds) {
    v = sum_row16(v);
    v = sum_rows4(v);
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

// A row's pieces i = t, t + T, ... of E floats (1 or 4); those past its end are 0.
template <int T, int N, int E>
struct Pieces {
    typedef float vec __attribute__((ext_vector_type(4)));
    float v[N][E];
    template <bool ONCE = false>
    __device__ __forceinline__ void load(const float *row, int t, int pieces) {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int i = t + k * T;
#pragma unroll
            for (int e = 0; e < E; e++) v[k][e] = 0.0f;
            if (i < pieces) {
                if constexpr (E == 4) {
                    const vec *at = reinterpret_cast<const vec *>(row + 4 * i);
                    const vec w = ONCE ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
                    for (int e = 0; e < E; e++) v[k][e] = w[e];
                } else {
                    v[k][0] = row[i];
                }
            }
        }
    }
    template <bool ONCE>
    __device__ __forceinline__ void store(float *row, int t, int pieces) const {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int i = t + k * T;
            if (i < pieces) {
                if constexpr (E == 4) {
                    vec *at = reinterpret_cast<vec *>(row + 4 * i);
                    const vec w = {v[k][0], v[k][1], v[k][2], v[k][3]};
                    if constexpr (ONCE)
                        __builtin_nontemporal_store(w, at);
                    else
                        *at = w;
                } else {
                    row[i] = v[k][0];
                }
            }
        }
    }
    __device__ __forceinline__ float squares() const {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < E; e++) s = fmaf(v[k][e], v[k][e], s);
        return s;
    }
};

// T threads a row, N pieces of E floats a thread. Everything that a row needs, its weights
// too, is asked for before the first sum: one round trip to memory and two sums are what a
// few rows cost. ONCE: the rows pass the caches by.
template <int T, int N, int E, bool ONCE>
__global__ __launch_bounds__(T < 256 ? 256 : T) void block_norm_kernel(const NormParams p) {
    constexpr int RPW = T < 256 ? 256 / T : 1;  // rows per workgroup
    __shared__ float lds[2][T / 64];
    const int t = threadIdx.x % T;
    const int pieces = p.dim / E;
    const int64_t r = (int64_t)blockIdx.x * RPW + threadIdx.x / T;
    if (r >= p.n_rows) return;  // (rows of one wave: a workgroup with rows of several holds one)
    Pieces<T, N, E> x, y, g, post, pre;
    x.template load<ONCE>(p.x + r * p.x_stride, t, pieces);
    if (p.y) y.template load<ONCE>(p.y + r * p.y_stride, t, pieces);
    if (p.post) post.load(p.post, t, pieces);
    if (p.gate) {
        if (ONCE && p.gate_stride)
            g.template load<ONCE>(p.gate + r * p.gate_stride, t, pieces);
        else
            g.load(p.gate + r * p.gate_stride, t, pieces);
    }
    if (p.norm_out) pre.load(p.pre, t, pieces);
    if (p.y) {
        float f = p.scale;
        if (p.post) f *= 1.0f / sqrtf(row_sum<T>(y.squares(), lds[0]) / (float)p.dim + p.eps);
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float z = y.v[k][e] * (p.gate ? g.v[k][e] * f : f);
                x.v[k][e] = p.post ? fmaf(z, post.v[k][e], x.v[k][e]) : x.v[k][e] + z;
            }
    }
    if (p.x_out) x.template store<ONCE>(p.x_out + r * p.x_out_stride, t, pieces);
    if (p.norm_out) {
        const float f = 1.0f / sqrtf(row_sum<T>(x.squares(), lds[1]) / (float)p.dim + p.eps);
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int e = 0; e < E; e++) x.v[k][e] *= f * pre.v[k][e];
        x.template store<ONCE>(p.norm_out + r * p.norm_out_stride, t, pieces);
    }
}

template <int T, int N, int E, bool ONCE = false>
int launch_as(gla_ctx *ctx, const NormParams &p) {
    constexpr int RPW = T < 256 ? 256 / T : 1;
    // (a grid holds fewer than 2^32 threads)
    constexpr int64_t kMost = (int64_t)1 << 21;
    for (int64_t r0 = 0; r0 < p.n_rows; r0 += kMost * RPW) {
        NormParams q = p;
        q.n_rows = (int)std::min<int64_t>(p.n_rows - r0, kMost * RPW);
        q.x += r0 * p.x_stride;
        if (q.y) q.y += r0 * p.y_stride;
        if (q.gate) q.gate += r0 * p.gate_stride;
        if (q.x_out) q.x_out += r0 * p.x_out_stride;
        if (q.norm_out) q.norm_out += r0 * p.norm_out_stride;
        hipLaunchKernelGGL((block_norm_kernel<T, N, E, ONCE>), dim3((unsigned)((q.n_rows + RPW - 1) / RPW)),
                           dim3(T < 256 ? 256 : T), 0, ctx->stream, q);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return set_error(GLA_ERR_KERNEL, "block_norm_kernel launch: %s", hipGetErrorString(e));
    }
    return GLA_OK;
}

template <int E>
int launch_e(gla_ctx *ctx, const NormParams &p) {
    const int pieces = p.dim / E;
    // Rows that are more than the last-level cache holds pass it by. us a call on rows that no
    // cache holds, past / through them: 7,993 rows of 4,096, all inputs (655 MB) 104 / 114,
    // without post and gate (524 MB) 91 / 96. Fewer go through them, for who wrote and who
    // reads them: inputs read past them on rows that they hold, 8,192 of 576 (75 MB) 16.9 / 13.1,
    // 256 of 4,096 (21 MB) 7.4 / 6.2.
    if constexpr (E == 4) {
        const int64_t rows = 1 + (p.y != nullptr) + (p.gate && p.gate_stride) + (p.x_out != nullptr) + (p.norm_out != nullptr);
        if (rows * p.n_rows * p.dim * 4 > (int64_t)256 << 20) {
            if (pieces <= 256) return launch_as<64, 4, 4, true>(ctx, p);
            if (pieces <= 1024) return launch_as<256, 4, 4, true>(ctx, p);
            return launch_as<1024, 4, 4, true>(ctx, p);
        }
    }
    if (pieces <= 64) return launch_as<64, 1, E>(ctx, p);
    if (pieces <= 256) return launch_as<64, 4, E>(ctx, p);
    // As many rows as the device has units, or fewer: the fewest loads a thread. More: several
    // workgroups a unit. us a captured call, 1,024 / 256 threads a row, both norms and a gate:
    // 64 rows of 3,584 4.25 / 4.43, 256 of 4,096 6.2 / 6.7, 7,993 of 4,096 118 / 113.
    if (pieces <= 1024 && p.n_rows <= ctx->n_cu) return launch_as<1024, 1, E>(ctx, p);
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
