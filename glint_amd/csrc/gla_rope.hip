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

constexpr int kMaxHeadDim = 256;
constexpr int kWaves = 4;   // waves of a workgroup, each on its own but for the sines of a shared row
constexpr int kAhead = 4;   // groups whose loads a wave has in flight
constexpr int kVByPage = 16;

// ---- rotating ------------------------------------------------------------------

struct Rope {
    const double *turns;
    int pairs;
    double amplitude;
};

// How a lane's 4 consecutive elements of a head find their pairs.
enum Mode {
    kCopy = 0,       // no rotation
    kAdjacent = 1,   // interleaved: in the lane's own registers
    kHalf = 2        // half: the partner is `pairs` elements away, in another lane's
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

// A wave's LDS: cos and sin of its row's pairs, then (kHalf) a group's heads.
__host__ __device__ constexpr size_t wave_lds(int mode, int pairs) {
    return mode == kCopy ? 0 : (size_t)pairs * sizeof(double2) + (mode == kHalf ? kMaxHeadDim * sizeof(float) : 0);
}

// cos and sin of pairs p0, p0 + step, ... at position pos: a lane evaluates one each
// and reads those that it needs from LDS (evaluations of a lane's own eight elements
// cost a call of one row 1.1 us of its 4.4).
__device__ __forceinline__ void turn_table(const Rope &r, double pos, double2 *table, int p0, int step) {
    for (int p = p0; p < r.pairs; p += step) {
        double2 t;
        cos_sin(pos * r.turns[p], r.amplitude, t.x, t.y);
        table[p] = t;
    }
}

// The factors of a lane's elements e0 .. e0 + 3 of a head; elements from
// 2 * pairs on are left alone.
template <int MODE, bool V>
struct Turn {
    static constexpr int N = MODE == kAdjacent ? 2 : 4;
    double c[N], s[N];
    const int pairs, e0, head_dim;
    float *stage;  // kHalf: the head's place in LDS, filled by the wave's lanes of this head

    __device__ __forceinline__ Turn(const Rope &r, int e0, int h, int head_dim, const double2 *table, float *wave_stage)
        : pairs(r.pairs), e0(e0), head_dim(head_dim) {
        if constexpr (MODE != kCopy) {
            stage = wave_stage + h * head_dim;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int e = MODE == kAdjacent ? e0 / 2 + j : e0 + j;
                const bool second = MODE == kHalf && e >= r.pairs;
                const double2 t = table[min(second ? e - r.pairs : e, r.pairs - 1)];
                c[j] = t.x;
                s[j] = MODE == kHalf && !second ? -t.y : t.y;
            }
        }
    }

    __device__ __forceinline__ void apply(float (&x)[4]) const {
        if constexpr (MODE == kAdjacent) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const double a = x[2 * j], b = x[2 * j + 1];
                if (e0 / 2 + j < pairs) {
                    x[2 * j] = (float)fma(a, c[j], -(b * s[j]));
                    x[2 * j + 1] = (float)fma(a, s[j], b * c[j]);
                }
            }
        } else if constexpr (MODE == kHalf) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the last head's reads
            if constexpr (V) {
                *reinterpret_cast<float4 *>(stage + e0) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (e0 + j < head_dim) stage[e0 + j] = x[j];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (V && pairs % 4 == 0) {  // the four are of one half, their partners together
                if (e0 < 2 * pairs) {
                    const float4 b = *reinterpret_cast<const float4 *>(stage + (e0 < pairs ? e0 + pairs : e0 - pairs));
                    x[0] = (float)fma((double)x[0], c[0], (double)b.x * s[0]);
                    x[1] = (float)fma((double)x[1], c[1], (double)b.y * s[1]);
                    x[2] = (float)fma((double)x[2], c[2], (double)b.z * s[2]);
                    x[3] = (float)fma((double)x[3], c[3], (double)b.w * s[3]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int e = e0 + j;
                    if (e < 2 * pairs) {
                        const double b = stage[e < pairs ? e + pairs : e - pairs];
                        x[j] = (float)fma((double)x[j], c[j], b * s[j]);
                    }
                }
            }
        }
    }
};

// 4 elements of a head, `n` of them inside it (at least one); V: all 4, 16-byte aligned
template <bool V>
__device__ __forceinline__ void load4(float (&x)[4], const float *p, int n) {
    if constexpr (V) {
        const float4 a = *reinterpret_cast<const float4 *>(p);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = j < n ? p[j] : 0.0f;
    }
}
template <bool V>
__device__ __forceinline__ void store4(float *p, const float (&x)[4], int n) {
    if constexpr (V) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < n) p[j] = x[j];
    }
}

// Groups g0 .. g1 - 1 through load(x, g) and then use(x, g), kAhead loads in flight.
template <class Load, class Use>
__device__ __forceinline__ void stream_groups(float (&x)[kAhead][4], int g0, int g1, const Load &load, const Use &use) {
    for (int g = g0; g < g1; g += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (g + i >= g1) break;
            float e[4] = {x[i][0], x[i][1], x[i][2], x[i][3]};
            if (g + i + kAhead < g1) load(x[i], g + i + kAhead);
            use(e, g + i);
        }
    }
}

// A wave takes heads of one row: `lanes` = ceil(head_dim / 4) lanes a head,
// 64 / lanes heads (a group) at a time. Bound: memory for many rows (7,993 rows
// of 32 x 128, 262 MB, at the rate of a large copy), launch and latency for few.
template <int MODE, bool V>
__global__ __launch_bounds__(kWaves * 64) void rope_rows_kernel(const Rope r, const float *x, int64_t x_stride,
                                                                float *out, int64_t out_stride, int n_rows,
                                                                int n_heads, int head_dim, int lanes, int parts,
                                                                const int32_t *pos) {
    extern __shared__ double2 lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t item = blockIdx.x * kWaves + wave;
    const int row = (int)(item / (uint32_t)parts);
    const int part = (int)(item - (uint32_t)row * parts);
    if (row >= n_rows) return;
    const int per = 64 / lanes;  // heads at a time
    // lanes past the last whole head repeat its first one's work (they take part
    // in the pairs' evaluation) and store nothing
    const bool spare = lane >= per * lanes;
    const int h = spare ? per - 1 : lane / lanes;
    const int e0 = spare ? 0 : (lane - h * lanes) * 4;
    const int groups = (n_heads + per - 1) / per;
    const int g0 = (int)((int64_t)groups * part / parts), g1 = (int)((int64_t)groups * (part + 1) / parts);
    const float *src = x + row * x_stride + e0;
    float *dst = out + row * out_stride + e0;
    const auto load = [&](float (&e)[4], int g) {
        load4<V>(e, src + (int64_t)min(g * per + h, n_heads - 1) * head_dim, head_dim - e0);
    };
    float ring[kAhead][4];
#pragma unroll
    for (int i = 0; i < kAhead; i++)
        if (g0 + i < g1) load(ring[i], g0 + i);
    double2 *table = lds + wave * (wave_lds(MODE, r.pairs) / sizeof(double2));
    turn_table(r, (double)pos[row], table, lane, 64);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const Turn<MODE, V> t(r, e0, h, head_dim, table, reinterpret_cast<float *>(table + r.pairs));
    stream_groups(ring, g0, g1, load, [&](float (&e)[4], int g) {
        t.apply(e);
        const int head = g * per + h;
        if (head < n_heads && !spare) store4<V>(dst + (int64_t)head * head_dim, e, head_dim - e0);
    });
}

// ---- append ---------------------------------------------------------------------

struct Append {
    RowOps o;
    PageMap pm;
    Rope rope;
    const int32_t *q_start, *pos_offset;
    int n_seqs, max_q_len, parts;
    int row_blocks;  // blocks of a sequence that take rows; the others take pages of V
    int v_by_page;
    const float *k, *v, *q;
    float *q_out;
    int64_t k_stride, v_stride, q_stride;
    int n_heads, n_kv;
};

constexpr int kMaxGridY = 32768;  // sequences along y, the rest along z
constexpr int kMaxSeqs = kMaxGridY * 65535;  // a launch's limit along z

// The storage page of (b, page lp of the sequence), or -1 where there is none.
__device__ __forceinline__ int64_t storage_page(const PageMap &pm, int b, int64_t lp) {
    int64_t page;
    if (pm.page_table) {
        page = pm.page_table[(int64_t)b * pm.pt_stride + lp];
    } else {
        const int s = pm.seq_slot ? pm.seq_slot[b] : b;
        if (s < 0 || s >= pm.n_slots) return -1;
        page = (int64_t)s * pm.seq_page_stride + pm.layer_page_off + lp;
    }
    return page < 0 || page >= pm.n_pages ? -1 : page;
}

// Maximum over the 16 lanes of a row: rotations by 8, 4, 2 and 1.
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xf, 0xf, true)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x124, 0xf, 0xf, true)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x122, 0xf, 0xf, true)));
    return fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x121, 0xf, 0xf, true)));
}

// V of a Q8_0 page: a wave takes 64 dimensions of one head's 16 positions, the
// kilobyte that lies together in the page (q8v_off), so lane (sg, j) makes the 16
// bytes of positions 4 sg .. +3 and dimensions j, j + 16, j + 32, j + 48 and
// stores them at once; row by row each byte is a store of its own (6,570 ragged rows
// with their q and read back 122 us, page by page and with shared sines 96). Positions of
// the page that are not new stay: a group of four with such is stored byte by byte.
__device__ __forceinline__ void append_v_page(const Append &a, int b, int idx, int lane) {
    const int pieces = a.o.head_dim >> 6;
    const int piece = idx % pieces;
    const int head = idx / pieces % a.n_kv;
    const int chunk = idx / pieces / a.n_kv;
    const int first = a.q_start[b], last = a.q_start[b + 1];
    const int64_t p0 = a.pos_offset[b];
    const int64_t p1 = min(p0 + min(last - first, a.max_q_len), (int64_t)a.pm.pos_limit);
    const int64_t lp = (p0 >> 4) + chunk;
    if (p1 <= p0 || lp < 0 || lp * GLA_PAGE_SIZE >= p1) return;  // no new row in this page
    const int64_t page = storage_page(a.pm, b, lp);
    if (page < 0) return;
    const int sg = lane >> 4, j = lane & 15;
    const int64_t pos = lp * GLA_PAGE_SIZE + sg * 4;
    float x[4][4];
    bool in[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        in[i] = pos + i >= p0 && pos + i < p1;
        const float *src = a.v + (in[i] ? first + (pos + i - p0) : (int64_t)first) * a.v_stride + head * a.o.head_dim + piece * 64 + j;
#pragma unroll
        for (int c = 0; c < 4; c++) x[i][c] = src[c * 16];
    }
    int q[4][4];
    float scale = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int c2 = 0; c2 < 2; c2++) {  // the two blocks of 32 dimensions
            const float d = scale_of(row_max(fmaxf(fmaxf(0.0f, fabsf(x[i][2 * c2])), fabsf(x[i][2 * c2 + 1]))));
            const float inv = 1.0f / d;
            q[i][2 * c2] = quantize_one(x[i][2 * c2], inv);
            q[i][2 * c2 + 1] = quantize_one(x[i][2 * c2 + 1], inv);
            if (j == 2 * i + c2) scale = d;
        }
    uint32_t w[4];
#pragma unroll
    for (int c = 0; c < 4; c++) w[c] = quant_bytes(q[0][c], q[1][c], q[2][c], q[3][c]);
    uint8_t *dst = const_cast<uint8_t *>(a.o.L.v) + page * a.o.L.page_stride + head * a.o.L.head_stride + piece * 1024 +
                   lane * 16;
    if (in[0] && in[1] && in[2] && in[3]) {
        *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (in[i])
#pragma unroll
                for (int c = 0; c < 4; c++) dst[4 * c + i] = (uint8_t)(w[c] >> (8 * i));
    }
    // lane 2 i + c2 of a row of lanes holds the scale of position i, block c2
    const bool mine = j < 8 && pos + (j >> 1) >= p0 && pos + (j >> 1) < p1;
    if (mine) {
        uint8_t *vs = const_cast<uint8_t *>(a.o.L.vs) + page * a.o.L.page_stride + head * a.o.L.head_stride;
        reinterpret_cast<uint16_t *>(vs)[(sg * 4 + (j >> 1)) * (a.o.head_dim >> 5) + piece * 2 + (j & 1)] =
            __half_as_ushort(__float2half_rn(scale));
    }
}

// A wave takes a part of one new row: its groups of 64 * 4 elements are those
// of q, of K and (unless V goes page by page) of V in turn, head_dim / 4 lanes a
// head. Bound: memory for f32 prompts (6,144 rows of 48 x 128, 314 MB, 59.8 us, 5.2
// TB/s); the instructions that rotate in 64 bits and quantise, and K's stores of 8
// bytes a piece, for Q8_0 ones (264 MB, 56.6 us); launch and one chain of position,
// sine, quantise and store for single tokens (64 rows 5.0 us, a launch being 2.7).
template <int MODE, bool V>
__global__ __launch_bounds__(kWaves * 64) void kv_append_kernel(const Append a) {
    extern __shared__ double2 lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int b = blockIdx.z * kMaxGridY + blockIdx.y;
    if (b >= a.n_seqs) return;
    if ((int)blockIdx.x >= a.row_blocks) {
        append_v_page(a, b, (blockIdx.x - a.row_blocks) * kWaves + wave, lane);
        return;
    }
    // Workgroups go round the eight XCDs; of a Q8_0 storage 16 rows at a time go to one,
    // whose L2 then puts the 8-byte pieces of their K together (6,570 ragged rows 63.4 ->
    // 61.4 us).
    uint32_t block = blockIdx.x;
    if (a.o.q8) {
        const uint32_t page = GLA_PAGE_SIZE / kWaves * a.parts, at = block / (8 * page) * (8 * page), o = block - at;
        if (at + 8 * page <= (uint32_t)a.row_blocks) block = at + o % 8 * page + o / 8;
    }
    const uint32_t item = block * kWaves + wave;
    const int i = (int)(item / (uint32_t)a.parts);
    const int part = (int)(item - (uint32_t)i * a.parts);
    const int first = a.q_start[b], last = a.q_start[b + 1];
    if (i >= min(last - first, a.max_q_len)) return;
    const int64_t r = (int64_t)first + i;
    const int64_t pos = (int64_t)a.pos_offset[b] + i;

    const int head_dim = a.o.head_dim;
    const int lanes = head_dim >> 2, per = 64 / lanes;
    const int h = lane / lanes;
    const int e0 = (lane - h * lanes) * 4;
    const int gq = a.q ? (a.n_heads + per - 1) / per : 0, gk = (a.n_kv + per - 1) / per;
    const int groups = gq + (a.v_by_page ? gk : 2 * gk);
    const int g0 = (int)((int64_t)groups * part / a.parts), g1 = (int)((int64_t)groups * (part + 1) / a.parts);
    const auto load = [&](float (&e)[4], int g) {
        const float *src;
        if (g < gq) {
            src = a.q + r * a.q_stride + min(g * per + h, a.n_heads - 1) * head_dim;
        } else {
            const bool v = g >= gq + gk;
            const int head = min((g - gq - (v ? gk : 0)) * per + h, a.n_kv - 1);
            src = (v ? a.v + r * a.v_stride : a.k + r * a.k_stride) + head * head_dim;
        }
        load4<V>(e, src + e0, 4);
    };
    float ring[kAhead][4];
#pragma unroll
    for (int n = 0; n < kAhead; n++)
        if (g0 + n < g1) load(ring[n], g0 + n);
    int64_t row = -1;
    if (g1 > gq && pos >= 0 && pos < a.pm.pos_limit) {
        const int64_t page = storage_page(a.pm, b, pos >> 4);
        if (page >= 0) row = page * GLA_PAGE_SIZE + (pos & 15);
    }
    const auto rest = [&](const auto &t) {
        stream_groups(ring, g0, g1, load, [&](float (&e)[4], int g) {
            if (g < gq + gk) t.apply(e);
            if (g < gq) {
                const int head = g * per + h;
                if (head < a.n_heads) store4<V>(a.q_out + (r * a.n_heads + head) * head_dim + e0, e, 4);
                return;
            }
            const int which = g >= gq + gk;
            const int head = (g - gq - which * gk) * per + h;
            if (head >= a.n_kv || row < 0) return;
            const int gi = head * head_dim + e0;
            if (a.o.q8)
                store_q8(a.o, row, gi, which, e);
            else
                store4<true>(reinterpret_cast<float *>(const_cast<uint8_t *>(which ? a.o.L.v : a.o.L.k) +
                                                       elem_off(a.o, row, gi, 4)), e, 4);
        });
    };
    double2 *own = lds + wave * (wave_lds(MODE, a.rope.pairs) / sizeof(double2)), *table = own;
    if constexpr (MODE != kCopy) {
        if (a.parts % kWaves == 0) {  // the workgroup's waves have one row
            table = lds;
            turn_table(a.rope, (double)pos, table, threadIdx.x, kWaves * 64);
            __syncthreads();
        } else if (g0 < gq + gk) {
            turn_table(a.rope, (double)pos, table, lane, 64);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
    if (MODE == kCopy || g0 >= gq + gk)
        rest(Turn<kCopy, V>(a.rope, e0, h, head_dim, nullptr, nullptr));
    else
        rest(Turn<MODE, V>(a.rope, e0, h, head_dim, table, reinterpret_cast<float *>(own + a.rope.pairs)));
}

bool aligned16(const void *p, int64_t stride) { return ((uintptr_t)p & 15) == 0 && stride % 4 == 0; }

int check_plan(const gla_ctx *ctx, const gla_rope_plan *r, const char *fn) {
    if (r->ctx != ctx)
        return set_error(GLA_ERR_INVALID, "%s: the rotary plan belongs to %s", fn,
                         r->ctx ? "another context" : "a destroyed context");
    return GLA_OK;
}

Rope rope_of(const gla_rope_plan *p) { return Rope{p->turns, p->pairs, p->amplitude}; }

// Parts of a row's `groups` that waves take: about `waves` of them in all, at
// most one group each. Short waves keep the last round of a long call short;
// waves of rows that ragged sequences do not have cost an append a little. us:
// 7,993 query rows, 4,096 / 16,384 / 32,768 / 65,536 / 131,072 waves 55.3 / 51.6 /
// 50.3 / 49.5 / 48.9; appends, 6,000 / 16,384 / 24,576: 6,570 ragged rows into a Q8_0
// pool 65.5 / 61.5 / 61.4, 6,144 of one length 60.4 / 56.4 / 56.9, 7,968 ragged f32
// ones 82.9 / 79.9 / 79.6.
constexpr int kRopeWaves = 65536, kAppendWaves = 24576;
int parts_of(int64_t rows, int groups, int waves) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(groups, (waves + rows - 1) / rows));
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
    const int lanes = (d + 3) / 4, per = 64 / lanes;
    const int parts = parts_of(n_rows, (n_heads + per - 1) / per, kRopeWaves);
    const int64_t blocks = ((int64_t)n_rows * parts + kWaves - 1) / kWaves;
    GLA_REQUIRE(blocks <= INT32_MAX / (kWaves * 64), "gla_rope_rows: %d rows are too many for one call", n_rows);
    const bool vec = d % 4 == 0 && aligned16(x, x_stride) && aligned16(out, out_stride);
    auto kernel = plan->half ? (vec ? rope_rows_kernel<kHalf, true> : rope_rows_kernel<kHalf, false>)
                             : (vec ? rope_rows_kernel<kAdjacent, true> : rope_rows_kernel<kAdjacent, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kWaves * 64), kWaves * wave_lds(plan->half ? kHalf : kAdjacent, plan->pairs),
                       ctx->stream, rope_of(plan), x, x_stride, out, out_stride, n_rows, n_heads, d, lanes, parts, pos);
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
    GLA_REQUIRE(a->n_seqs >= 0 && a->n_seqs <= kMaxSeqs && a->max_q_len >= 0,
                "gla_kv_append: n_seqs %d (0 to %d), max_q_len %d", a->n_seqs, kMaxSeqs, a->max_q_len);
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
    // V of a Q8_0 storage page by page where a sequence's rows fill pages, else
    // with its row
    p.v_by_page = p.o.q8 && p.max_q_len >= kVByPage;
    const int per = 64 / (kv->head_dim / 4);
    const int gk = (p.n_kv + per - 1) / per;
    const int groups = (a->q ? (a->n_heads + per - 1) / per : 0) + (p.v_by_page ? gk : 2 * gk);
    p.parts = parts_of((int64_t)a->n_seqs * a->max_q_len, groups, kAppendWaves);
    const int64_t row_blocks = ((int64_t)p.max_q_len * p.parts + kWaves - 1) / kWaves;
    const int64_t chunks = ((int64_t)p.max_q_len + GLA_PAGE_SIZE - 2) / GLA_PAGE_SIZE + 1;  // pages a sequence may touch
    const int64_t v_blocks = p.v_by_page ? (chunks * p.n_kv * (kv->head_dim / 64) + kWaves - 1) / kWaves : 0;
    GLA_REQUIRE(row_blocks + v_blocks <= INT32_MAX / (kWaves * 64), "gla_kv_append: sequences of %d rows are too long for one call",
                a->max_q_len);
    p.row_blocks = (int)row_blocks;
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    const bool vec = aligned16(p.k, p.k_stride) && aligned16(p.v, p.v_stride) &&
                     (!p.q || (aligned16(p.q, p.q_stride) && aligned16(p.q_out, 0)));
    int mode = kCopy;
    auto kernel = vec ? kv_append_kernel<kCopy, true> : kv_append_kernel<kCopy, false>;
    if (a->rope) {
        mode = a->rope->half ? kHalf : kAdjacent;
        kernel = a->rope->half ? (vec ? kv_append_kernel<kHalf, true> : kv_append_kernel<kHalf, false>)
                               : (vec ? kv_append_kernel<kAdjacent, true> : kv_append_kernel<kAdjacent, false>);
    }
    const dim3 grid((unsigned)(row_blocks + v_blocks), std::min(a->n_seqs, kMaxGridY), (a->n_seqs + kMaxGridY - 1) / kMaxGridY);
    hipLaunchKernelGGL(kernel, grid, dim3(kWaves * 64), kWaves * wave_lds(mode, p.rope.pairs), ctx->stream, p);
    return launched("kv_append_kernel");
    GLA_GUARD_END
}

}  // extern "C"
