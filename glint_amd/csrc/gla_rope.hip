// gla_rope.hip -- rotary positions (both layouts, part of the head, stretched
// frequencies) and the append that rotates K and q on the way from a projection
// into a storage.
//
// A pair (a, b) at position pos turns by the angle pos * f: (a c - b s,
// a s + b c), c and s the amplitude times cos and sin. The angle is taken in
// turns, t = pos * (f / 2 pi), and reduced exactly: r = t - round(t), then the
// octant round(4 r) and y = r - octant / 4 in [-1/8, 1/8], whose sine and
// cosine are the Taylor series of 2 pi y to z^15 and z^16 (the next terms are
// below 2^-53). All of it is 64-bit: a far position's angle keeps its digits,
// and a value is rounded once, so a Q8_0 quant is the one that the exactly
// rotated value has. FP64 runs at the rate of unpacked FP32 on this part, and
// one evaluation serves every head of a row.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <vector>

#include "gla_rows.h"

struct gla_rope_plan {
    gla_ctx *ctx = nullptr;
    int head_dim = 0;
    int pairs = 0;
    bool half = false;
    double amplitude = 1.0;
    double *turns = nullptr;  // device [pairs]: turns per position
};

namespace gla {

void detach_rope(gla_rope_plan *r) {
    if (r->turns) (void)hipFree(r->turns);
    r->turns = nullptr;
    r->ctx = nullptr;
}

namespace {

constexpr int kMaxHeadDim = 512;

// ---- rotating ------------------------------------------------------------------

struct Rope {
    const double *turns;
    int pairs;
    double amplitude;
};

// How a lane's 8 consecutive elements of a head find their pairs.
enum Mode {
    kCopy = 0,       // no rotation
    kAdjacent = 1,   // interleaved: in the lane's own registers
    kHalf = 2        // half: the partner is pairs elements away, in another lane's
};

__device__ __forceinline__ void cos_sin(double t, double amp, double &c, double &s) {
    const double r = t - rint(t);
    const double o = rint(4.0 * r);
    const double z = fma(o, -0.25, r) * 6.283185307179586476925286766559;
    const double u = z * z;
    double a = -1.0 / 1307674368000.0;  // 15!
    a = fma(a, u, 1.0 / 6227020800.0);
    a = fma(a, u, -1.0 / 39916800.0);
    a = fma(a, u, 1.0 / 362880.0);
    a = fma(a, u, -1.0 / 5040.0);
    a = fma(a, u, 1.0 / 120.0);
    a = fma(a, u, -1.0 / 6.0);
    a = fma(a * u, z, z);
    double b = 1.0 / 20922789888000.0;  // 16!
    b = fma(b, u, -1.0 / 87178291200.0);
    b = fma(b, u, 1.0 / 479001600.0);
    b = fma(b, u, -1.0 / 3628800.0);
    b = fma(b, u, 1.0 / 40320.0);
    b = fma(b, u, -1.0 / 720.0);
    b = fma(b, u, 1.0 / 24.0);
    b = fma(b, u, -0.5);
    b = fma(b, u, 1.0);
    const int q = (int)o & 3;  // quarter turns
    const double cc = (q & 1) ? a : b, ss = (q & 1) ? b : a;
    c = (q == 1 || q == 2) ? -cc * amp : cc * amp;
    s = (q == 2 || q == 3) ? -ss * amp : ss * amp;
}

// The factors of a lane's elements e0 .. e0 + 7: x -> own * c + partner * s.
template <int MODE>
struct Turn {
    double c[MODE == kAdjacent ? 4 : 8], s[MODE == kAdjacent ? 4 : 8];

    __device__ __forceinline__ void set(const Rope &r, int e0, double pos) {
        if constexpr (MODE == kAdjacent) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int p = e0 / 2 + j;
                if (p < r.pairs) cos_sin(pos * r.turns[p], r.amplitude, c[j], s[j]);
            }
        } else if constexpr (MODE == kHalf) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int e = e0 + j;
                if (e < 2 * r.pairs) {
                    const bool second = e >= r.pairs;
                    cos_sin(pos * r.turns[second ? e - r.pairs : e], r.amplitude, c[j], s[j]);
                    if (!second) s[j] = -s[j];
                }
            }
        }
    }

    // x: elements e0 .. +7 of a head; `stage` the head's place in LDS (kHalf),
    // which the wave's lanes of this head fill together.
    __device__ __forceinline__ void apply(const Rope &r, int e0, int head_dim, float (&x)[8], float *stage) const {
        if constexpr (MODE == kAdjacent) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const double a = x[2 * j], b = x[2 * j + 1];
                if (e0 / 2 + j < r.pairs) {
                    x[2 * j] = (float)fma(a, c[j], -(b * s[j]));
                    x[2 * j + 1] = (float)fma(a, s[j], b * c[j]);
                }
            }
        } else if constexpr (MODE == kHalf) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the last head's reads
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (e0 + j < head_dim) stage[e0 + j] = x[j];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int e = e0 + j;
                if (e < 2 * r.pairs) {
                    const double b = stage[e < r.pairs ? e + r.pairs : e - r.pairs];
                    x[j] = (float)fma((double)x[j], c[j], b * s[j]);
                }
            }
        }
    }
};

// 8 elements of a head, `n` of them inside it (at least one); V: all 8, 16-byte aligned
template <bool V>
__device__ __forceinline__ void load8(float (&x)[8], const float *p, int n) {
    if constexpr (V) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = j < n ? p[j] : 0.0f;
    }
}
template <bool V>
__device__ __forceinline__ void store8(float *p, const float (&x)[8], int n) {
    if constexpr (V) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < n) p[j] = x[j];
    }
}

constexpr int kWaves = 4;

// A wave takes heads of one row: `lanes` = ceil(head_dim / 8) lanes a head,
// 64 / lanes heads at a time.
template <int MODE, bool V>
__global__ __launch_bounds__(kWaves * 64) void rope_rows_kernel(const Rope r, const float *x, int64_t x_stride,
                                                                float *out, int64_t out_stride, int n_rows,
                                                                int n_heads, int head_dim, int lanes, int parts,
                                                                const int32_t *pos) {
    __shared__ __attribute__((aligned(16))) float lds[kWaves][kMaxHeadDim];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * kWaves + wave;
    const int64_t row = item / parts;
    const int part = (int)(item - row * parts);
    if (row >= n_rows) return;
    const int per = 64 / lanes;  // heads at a time
    const int h = lane / lanes;
    if (h >= per) return;
    const int e0 = (lane - h * lanes) * 8;
    const int groups = (n_heads + per - 1) / per;
    const int g0 = (int)((int64_t)groups * part / parts), g1 = (int)((int64_t)groups * (part + 1) / parts);
    Turn<MODE> t;
    t.set(r, e0, pos[row]);
    for (int g = g0; g < g1; g++) {
        const int head = g * per + h;
        if (head >= n_heads) continue;
        float e[8];
        load8<V>(e, x + row * x_stride + (int64_t)head * head_dim + e0, head_dim - e0);
        t.apply(r, e0, head_dim, e, lds[wave] + h * head_dim);
        store8<V>(out + row * out_stride + (int64_t)head * head_dim + e0, e, head_dim - e0);
    }
}

// ---- append ---------------------------------------------------------------------

struct Append {
    RowOps o;
    PageMap pm;
    Rope rope;
    const int32_t *q_start, *pos_offset;
    int n_seqs, max_q_len, parts;
    const float *k, *v, *q;
    float *q_out;
    int64_t k_stride, v_stride, q_stride;
    int n_heads, n_kv;
};

// The storage row of (b, pos), or -1 where there is none.
__device__ __forceinline__ int64_t storage_row(const PageMap &pm, int b, int64_t pos) {
    if (pos < 0 || pos >= pm.pos_limit) return -1;
    int64_t page;
    if (pm.page_table) {
        page = pm.page_table[(int64_t)b * pm.pt_stride + (pos >> 4)];
    } else {
        const int s = pm.seq_slot ? pm.seq_slot[b] : b;
        if (s < 0 || s >= pm.n_slots) return -1;
        page = (int64_t)s * pm.seq_page_stride + pm.layer_page_off + (pos >> 4);
    }
    return page < 0 || page >= pm.n_pages ? -1 : page * GLA_PAGE_SIZE + (pos & 15);
}

// A wave takes a part of one new row: its groups of 64 * 8 elements are those
// of q, of K and of V in turn (head_dim / 8 lanes a head).
template <int MODE, bool V>
__global__ __launch_bounds__(kWaves * 64) void kv_append_kernel(const Append a) {
    __shared__ __attribute__((aligned(16))) float lds[kWaves][kMaxHeadDim];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * kWaves + wave;
    const int64_t place = item / a.parts;
    const int part = (int)(item - place * a.parts);
    const int b = (int)(place / a.max_q_len);
    const int i = (int)(place - (int64_t)b * a.max_q_len);
    if (b >= a.n_seqs) return;
    const int first = a.q_start[b], last = a.q_start[b + 1];
    if (i >= last - first) return;
    const int64_t r = (int64_t)first + i;
    const int64_t pos = (int64_t)a.pos_offset[b] + i;
    const int64_t row = storage_row(a.pm, b, pos);

    const int head_dim = a.o.head_dim;
    const int lanes = head_dim >> 3, per = 64 / lanes;
    const int h = lane / lanes;
    const int e0 = (lane - h * lanes) * 8;
    const int gq = a.q ? (a.n_heads + per - 1) / per : 0, gk = (a.n_kv + per - 1) / per;
    const int groups = gq + 2 * gk;
    const int g0 = (int)((int64_t)groups * part / a.parts), g1 = (int)((int64_t)groups * (part + 1) / a.parts);
    Turn<MODE> t;
    if (MODE != kCopy && g0 < gq + gk) t.set(a.rope, e0, (double)pos);
    for (int g = g0; g < g1; g++) {
        float e[8];
        if (g < gq) {
            const int head = g * per + h;
            if (head >= a.n_heads) continue;
            load8<V>(e, a.q + r * a.q_stride + head * head_dim + e0, 8);
            t.apply(a.rope, e0, head_dim, e, lds[wave] + h * head_dim);
            store8<V>(a.q_out + (r * a.n_heads + head) * head_dim + e0, e, 8);
            continue;
        }
        const int which = g >= gq + gk;
        const int head = (g - gq - which * gk) * per + h;
        if (head >= a.n_kv || row < 0) continue;
        const int gi = head * head_dim + e0;
        load8<V>(e, which ? a.v + r * a.v_stride + gi : a.k + r * a.k_stride + gi, 8);
        if (!which) t.apply(a.rope, e0, head_dim, e, lds[wave] + h * head_dim);
        if (a.o.q8)
            store_q8(a.o, row, gi, which, e);
        else
            store8<true>(reinterpret_cast<float *>(const_cast<uint8_t *>(which ? a.o.L.v : a.o.L.k) +
                                                   elem_off(a.o, row, gi, 4)), e, 8);
    }
}

bool aligned16(const void *p, int64_t stride) { return ((uintptr_t)p & 15) == 0 && stride % 4 == 0; }

int check_plan(const gla_ctx *ctx, const gla_rope_plan *r, const char *fn) {
    if (r->ctx != ctx)
        return set_error(GLA_ERR_INVALID, "%s: the rotary plan belongs to %s", fn,
                         r->ctx ? "another context" : "a destroyed context");
    return GLA_OK;
}

Rope rope_of(const gla_rope_plan *p) { return Rope{p->turns, p->pairs, p->amplitude}; }

// Parts of a row's `groups` that waves take: enough waves to fill the chip's
// 1,024 SIMDs a few times over, at most one group each.
int parts_of(int64_t rows, int groups) {
    const int64_t want = (4096 + rows - 1) / rows;
    return (int)std::max<int64_t>(1, std::min<int64_t>(groups, want));
}

// The frequencies and the amplitude of a specification, or an error.
int frequencies(const gla_rope_spec *s, std::vector<double> *freq, double *amplitude) {
    const char *fn = "gla_rope_spec";
    GLA_REQUIRE(s, "%s: NULL argument", fn);
    GLA_REQUIRE(s->head_dim >= 1 && s->head_dim <= kMaxHeadDim, "%s: head_dim %d (supported: 1 to %d)", fn, s->head_dim,
                kMaxHeadDim);
    const int rot = s->rot_dim ? s->rot_dim : s->head_dim;
    GLA_REQUIRE(rot > 0 && rot % 2 == 0 && rot <= s->head_dim, "%s: rot_dim %d is not an even part of head_dim %d", fn,
                rot, s->head_dim);
    GLA_REQUIRE(s->freq_dim >= 0, "%s: freq_dim %d < 0", fn, s->freq_dim);
    GLA_REQUIRE(s->layout == GLA_ROPE_INTERLEAVED || s->layout == GLA_ROPE_HALF, "%s: bad layout %d", fn, (int)s->layout);
    GLA_REQUIRE(s->scaling >= GLA_ROPE_NONE && s->scaling <= GLA_ROPE_YARN, "%s: bad scaling %d", fn, (int)s->scaling);
    GLA_REQUIRE(isfinite(s->freq_base) && s->freq_base > 0, "%s: freq_base %g", fn, s->freq_base);
    GLA_REQUIRE(isfinite(s->amplitude) && s->amplitude >= 0, "%s: amplitude %g", fn, s->amplitude);
    const bool stretched = s->scaling != GLA_ROPE_NONE;
    const bool banded = s->scaling == GLA_ROPE_BANDS || s->scaling == GLA_ROPE_YARN;
    GLA_REQUIRE(!stretched || (isfinite(s->factor) && s->factor > 0), "%s: factor %g", fn, s->factor);
    GLA_REQUIRE(!banded || s->original_ctx > 0, "%s: original_ctx %d", fn, s->original_ctx);
    GLA_REQUIRE(!banded || (isfinite(s->high) && s->low > 0 && s->low < s->high), "%s: low %g, high %g", fn, s->low, s->high);
    GLA_REQUIRE(s->scaling != GLA_ROPE_YARN || s->freq_base != 1.0, "%s: freq_base 1 has no turns to tell pairs by", fn);
    const int fd = s->freq_dim ? s->freq_dim : rot;
    const double two_pi = 2.0 * M_PI;
    double first = 0.0, last = 0.0;
    if (s->scaling == GLA_ROPE_YARN) {
        const auto pair_of = [&](double t) { return fd * log(s->original_ctx / (two_pi * t)) / (2.0 * log(s->freq_base)); };
        first = std::max(floor(pair_of(s->high)), 0.0);
        last = std::min(ceil(pair_of(s->low)), fd - 1.0);
        last = first + std::max(last - first, 0.001);
    }
    freq->resize(rot / 2);
    for (int p = 0; p < rot / 2; p++) {
        double g = pow(s->freq_base, -2.0 * p / fd);
        if (s->divisors) {
            GLA_REQUIRE(isfinite(s->divisors[p]) && s->divisors[p] != 0.0f, "%s: divisor %d is %g", fn, p,
                        (double)s->divisors[p]);
            g /= s->divisors[p];
        }
        double keep = 1.0;
        if (s->scaling == GLA_ROPE_LINEAR)
            keep = 0.0;
        else if (s->scaling == GLA_ROPE_BANDS)
            keep = (s->original_ctx * g / two_pi - s->low) / (s->high - s->low);
        else if (s->scaling == GLA_ROPE_YARN)
            keep = 1.0 - (p - first) / (last - first);
        keep = std::min(1.0, std::max(0.0, keep));
        const double f = stretched ? (1.0 - keep) * (g / s->factor) + keep * g : g;
        GLA_REQUIRE(isfinite(f), "%s: the frequency of pair %d is not finite", fn, p);
        (*freq)[p] = f;
    }
    *amplitude = s->amplitude > 0 ? s->amplitude
                 : s->scaling == GLA_ROPE_YARN && s->factor > 1 ? 0.1 * log(s->factor) + 1.0
                                                                : 1.0;
    return GLA_OK;
}

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GLA_OK : set_error(GLA_ERR_KERNEL, "%s launch: %s", what, hipGetErrorString(e));
}

}  // namespace
}  // namespace gla

using namespace gla;

extern "C" {

int gla_rope_freqs(const gla_rope_spec *spec, double *freqs, double *amplitude) {
    GLA_GUARD_BEGIN
    std::vector<double> f;
    double amp = 1.0;
    if (int rc = frequencies(spec, &f, &amp)) return rc;
    if (freqs) memcpy(freqs, f.data(), f.size() * sizeof(double));
    if (amplitude) *amplitude = amp;
    return GLA_OK;
    GLA_GUARD_END
}

int gla_rope_plan_create(gla_ctx *ctx, const gla_rope_spec *spec, gla_rope_plan **out) {
    GLA_GUARD_BEGIN
    GLA_REQUIRE(ctx && spec && out, "gla_rope_plan_create: NULL argument");
    *out = nullptr;
    std::vector<double> f;
    double amp = 1.0;
    if (int rc = frequencies(spec, &f, &amp)) return rc;
    for (double &x : f) x /= 2.0 * M_PI;
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    ctx->ropes.reserve(ctx->ropes.size() + 1);
    gla_rope_plan *p = new gla_rope_plan();
    p->ctx = ctx;
    p->head_dim = spec->head_dim;
    p->pairs = (int)f.size();
    p->half = spec->layout == GLA_ROPE_HALF;
    p->amplitude = amp;
    hipError_t e = hipMalloc(&p->turns, f.size() * sizeof(double));
    if (e == hipSuccess)
        e = hipMemcpyAsync(p->turns, f.data(), f.size() * sizeof(double), hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) {
        (void)hipGetLastError();  // not the next launch's
        if (p->turns) (void)hipFree(p->turns);
        delete p;
        return set_error(GLA_ERR_BUFFER, "gla_rope_plan_create: %s", hipGetErrorString(e));
    }
    ctx->ropes.push_back(p);
    *out = p;
    return GLA_OK;
    GLA_GUARD_END
}

int gla_rope_plan_destroy(gla_rope_plan *p) {
    GLA_GUARD_BEGIN
    if (!p) return GLA_OK;
    if (gla_ctx *ctx = p->ctx) {  // else its context already freed the frequencies
        (void)hipSetDevice(ctx->device);
        (void)hipStreamSynchronize(ctx->stream);
        ctx->ropes.erase(std::remove(ctx->ropes.begin(), ctx->ropes.end(), p), ctx->ropes.end());
        detach_rope(p);
    }
    delete p;
    return GLA_OK;
    GLA_GUARD_END
}

int gla_rope_rows(gla_ctx *ctx, const gla_rope_plan *plan, const float *x, int64_t x_stride, float *out,
                  int64_t out_stride, int n_rows, int n_heads, const int32_t *pos) {
    GLA_GUARD_BEGIN
    GLA_REQUIRE(ctx && plan, "gla_rope_rows: NULL argument");
    if (int rc = check_plan(ctx, plan, "gla_rope_rows")) return rc;
    GLA_REQUIRE(n_rows >= 0 && n_heads > 0, "gla_rope_rows: bad shape (rows %d, heads %d)", n_rows, n_heads);
    const int64_t width = (int64_t)n_heads * plan->head_dim;
    GLA_REQUIRE(width <= INT32_MAX, "gla_rope_rows: %d heads of %d", n_heads, plan->head_dim);
    if (!x_stride) x_stride = width;
    if (!out_stride) out_stride = width;
    GLA_REQUIRE(x_stride >= width && out_stride >= width, "gla_rope_rows: a stride is below the %lld floats of a row",
                (long long)width);
    if (n_rows == 0) return GLA_OK;
    GLA_REQUIRE(x && out && pos, "gla_rope_rows: NULL buffer");
    GLA_REQUIRE(x != out || x_stride == out_stride, "gla_rope_rows: in place needs one stride");
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    const int d = plan->head_dim;
    const int lanes = (d + 7) / 8, per = 64 / lanes;
    const int parts = parts_of(n_rows, (n_heads + per - 1) / per);
    const int64_t blocks = ((int64_t)n_rows * parts + kWaves - 1) / kWaves;
    GLA_REQUIRE(blocks <= INT32_MAX, "gla_rope_rows: %d rows are too many for one call", n_rows);
    const bool vec = d % 8 == 0 && aligned16(x, x_stride) && aligned16(out, out_stride);
    auto kernel = plan->half ? (vec ? rope_rows_kernel<kHalf, true> : rope_rows_kernel<kHalf, false>)
                             : (vec ? rope_rows_kernel<kAdjacent, true> : rope_rows_kernel<kAdjacent, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kWaves * 64), 0, ctx->stream, rope_of(plan), x, x_stride, out,
                       out_stride, n_rows, n_heads, d, lanes, parts, pos);
    return launched("rope_rows_kernel");
    GLA_GUARD_END
}

int gla_kv_append(gla_ctx *ctx, const gla_append_args *a) {
    GLA_GUARD_BEGIN
    GLA_REQUIRE(ctx && a && a->kv, "gla_kv_append: NULL argument");
    const gla_kv *kv = a->kv;
    if (int rc = check_owner(ctx, kv, "gla_kv_append")) return rc;
    if (a->rope) {
        if (int rc = check_plan(ctx, a->rope, "gla_kv_append")) return rc;
        GLA_REQUIRE(a->rope->head_dim == kv->head_dim, "gla_kv_append: the rotary plan is for heads of %d, the storage's are %d",
                    a->rope->head_dim, kv->head_dim);
    }
    GLA_REQUIRE(a->n_seqs >= 0 && a->max_q_len >= 0, "gla_kv_append: n_seqs %d, max_q_len %d", a->n_seqs, a->max_q_len);
    Append p;
    memset(&p, 0, sizeof(p));
    p.k_stride = a->k_stride ? a->k_stride : kv->kv_dim;
    p.v_stride = a->v_stride ? a->v_stride : kv->kv_dim;
    GLA_REQUIRE(p.k_stride >= kv->kv_dim && p.v_stride >= kv->kv_dim,
                "gla_kv_append: a stride is below the %d floats of a row", kv->kv_dim);
    if (a->q) {
        GLA_REQUIRE(a->n_heads > 0 && a->n_heads % kv->n_kv_heads == 0,
                    "gla_kv_append: n_heads %d is not a multiple of n_kv_heads %d", a->n_heads, kv->n_kv_heads);
        const int64_t width = (int64_t)a->n_heads * kv->head_dim;
        GLA_REQUIRE(width <= INT32_MAX, "gla_kv_append: %d heads of %d", a->n_heads, kv->head_dim);
        p.q_stride = a->q_stride ? a->q_stride : width;
        GLA_REQUIRE(p.q_stride >= width, "gla_kv_append: q_stride is below the %lld floats of a row", (long long)width);
        GLA_REQUIRE(a->q_out, "gla_kv_append: q without q_out");
        GLA_REQUIRE(a->q_out != a->q || p.q_stride == width, "gla_kv_append: q in place needs dense rows");
    }
    if (a->n_seqs == 0 || a->max_q_len == 0) return GLA_OK;
    GLA_REQUIRE(a->k && a->v && a->q_start && a->pos_offset, "gla_kv_append: NULL buffer");
    GLA_REQUIRE(a->page_table_stride <= INT32_MAX / GLA_PAGE_SIZE, "gla_kv_append: page_table_stride %d", a->page_table_stride);
    if (int rc = page_map_of(kv, a->layer, a->seq_slot, a->page_table, a->page_table_stride, &p.pm)) return rc;
    p.o = row_ops(kv);
    if (a->rope) p.rope = rope_of(a->rope);
    p.q_start = a->q_start;
    p.pos_offset = a->pos_offset;
    p.n_seqs = a->n_seqs;
    p.max_q_len = a->max_q_len;
    p.k = a->k;
    p.v = a->v;
    p.q = a->q;
    p.q_out = a->q_out;
    p.n_heads = a->n_heads;
    p.n_kv = kv->n_kv_heads;
    const int per = 64 / (kv->head_dim / 8);
    const int groups = (a->q ? (a->n_heads + per - 1) / per : 0) + 2 * ((p.n_kv + per - 1) / per);
    const int64_t places = (int64_t)a->n_seqs * a->max_q_len;
    p.parts = parts_of(places, groups);
    const int64_t blocks = (places * p.parts + kWaves - 1) / kWaves;
    GLA_REQUIRE(blocks <= INT32_MAX, "gla_kv_append: %d sequences of %d rows are too many for one call", a->n_seqs,
                a->max_q_len);
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    const bool vec = aligned16(p.k, p.k_stride) && aligned16(p.v, p.v_stride) &&
                     (!p.q || (aligned16(p.q, p.q_stride) && aligned16(p.q_out, 0)));
    auto kernel = vec ? kv_append_kernel<kCopy, true> : kv_append_kernel<kCopy, false>;
    if (a->rope)
        kernel = a->rope->half ? (vec ? kv_append_kernel<kHalf, true> : kv_append_kernel<kHalf, false>)
                               : (vec ? kv_append_kernel<kAdjacent, true> : kv_append_kernel<kAdjacent, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kWaves * 64), 0, ctx->stream, p);
    return launched("kv_append_kernel");
    GLA_GUARD_END
}

}  // extern "C"
