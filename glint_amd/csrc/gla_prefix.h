// gla_prefix.h -- the part of a batch's decode that groups of its sequences have
// in common (gfx950, matrix cores): the pages of a group's prefix, multiplied with the
// queries of all its rows at once.
//
// Math, of group g, KV head h and the 16 NT rows (sequence, query head of h) of a row
// tile, over a split of the prefix's pages:
//   S^T[key][row] = K . Q^T       s = cap(scale S) log2(e), -inf where a row does not see the key
//   m = max s, l = sum 2^(s - m), O^T[d][row] = V^T . P^T with P = 2^(s - m)
// (m, l, O) go to scratch, where the decode's combine kernel merges them with what the
// row has of its own.
//
// These workgroups run in one launch with those of the rows' own pages (Mixed), in the decode
// kernels of the two storages.
//
// Work: a wave takes a quarter of the split's pages by itself, operands straight from
// global memory into registers (the layouts of both storages are, or allow, the operand
// order), the next page's in flight while one is multiplied; the waves meet only to merge
// their (m, l, O) in LDS. Both products keep a row in a column of the tile: a lane's
// scores are the operand of the second product as they are, and a row's maximum is its
// four lanes'.
//
// What bounds it (whole calls, on clocks that have settled; the first some hundred after a pause
// are up to a tenth slower): Q8_0 vector issue (68% of the cycles, matrix 19%, in turn): 64 rows of
// 8-64 positions behind 8,192 at 32/8 heads, d = 128 43.4 us, 198 TFLOP/s of the attention's
// products, of 64-1,000 47.0; f32 the matrix rate from some 48 rows a group on (64 rows of 8-64 86.8
// us, 99 of the 138 TFLOP/s that a library product reaches), HBM and the tiles' re-reads before (24
// rows of 17-300 in 3 groups behind up to 4,096 at 16/8, d = 256 56.6 us, 252 MB, 4.5 TB/s).
// Two figures of a rule beside the code were taken in turn on one build, not always this one.
#pragma once

#include <math.h>

#include <algorithm>

#include "gla_internal.h"
#include "gla_lanes.h"

namespace gla {
namespace prefix {

using namespace lanes;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;

struct PrefixParams {
    KvLayout kv;
    PageMap pm;
    PrefixLaunch pre;
    const float *q;
    const int32_t *kv_start, *kv_len;  // of the batch's rows
    int max_kv_len;
    int n_seqs;
    int n_heads;
    int n_kv_heads;
    int group;
    float q_mul;    // scale (soft-cap) or scale * log2(e)
    float softcap;  // > 0: cap * tanh(s / cap)
    int columns;    // KV heads x row tiles of all groups
};

// x, for a rare block of code to start from: the block stays a branch, where the compiler
// would compute what is in it every time and select.
template <typename T>
__device__ __forceinline__ T rare(T x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The reference m of a row's exponents moves only when a score passes it by more than
// `lazy`: p is then at most 2^lazy, and most pages rescale nothing. f32 holds any p alike.
// Q8_0's pieces of p are halves, of which a row that lags wastes the top: p times the largest
// scale is below 2^14 for p = 1, as in the decode of single rows, and below 2^15.5 for the
// largest p (where m's unit rounds m + 1.5 to m + 2, at most 2^16 (1 - 2^-11), a half's largest).
// With 8 and 2^6 instead 2^-18 of the largest scale was off by 1e-3, and the calls were 1-2% faster.
constexpr float kLazy = 8.0f, kLazyQ8 = 1.5f;
// Moves m to the maximum of the row's four lanes where that passes it; what the sums are to be multiplied by.
__device__ __forceinline__ float moved(float &m, float mine, float lazy) {
    const float top = max_rows4(mine);
    const bool up = top > m + lazy;
    const float f = up ? fast_exp2(m - top) : 1.0f;
    m = up ? top : m;
    return f;
}

// A workgroup's place among the prefixes' (KV heads x row tiles of all groups, split, 0) or among
// those of the rows' own pages.
struct Place {
    int x, y, z;
};

// Row tile `at` of all groups': its group and its place among that group's tiles.
struct Tile {
    int group;  // < 0: there are not as many
    int at;
    int first, members;  // the group's rows, clamped into the batch
};
__device__ __forceinline__ Tile tile_of(const PrefixParams &p, int tile_rows, int at) {
    const int lane = threadIdx.x & 63;
    Tile t;
    t.group = -1;
    // (every wave by itself; a launch has fewer than 2^30 tiles, so that the sums stay in 32 bits)
    for (int i = 0, before = 0; i < p.pre.n_groups; i += 64) {
        const int g = min(i + lane, p.pre.n_groups - 1);
        const int first = min(max(p.pre.group_start[g], 0), p.n_seqs);
        const int members = min(max(min(p.pre.group_start[g + 1], p.n_seqs) - first, 0), p.pre.max_group);
        const int mine = i + lane < p.pre.n_groups ? (members * p.group + tile_rows - 1) / tile_rows : 0;
        const int end = before + sum_to_lane(mine);
        const uint64_t holds = __ballot(end > at);
        if (holds) {
            const int l = __builtin_ctzll(holds);
            t.group = i + l;
            t.at = at - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(mine, l));
            t.first = __builtin_amdgcn_readlane(first, l);
            t.members = __builtin_amdgcn_readlane(members, l);
            break;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return t;
}

// A wave's pages of a split's [from, to): its quarter of them (EVEN: taken two at a time).
struct Pages {
    int first, n;
};
template <bool EVEN>
__host__ __device__ __forceinline__ Pages wave_pages(int from, int to, int wave) {
    const int n = to > from ? to - from : 0;
    int each = (n + kWaves - 1) / kWaves;
    if (EVEN) each = (each + 1) & ~1;
    const int left = n - wave * each;
    return {from + wave * each, left < 0 ? 0 : (left < each ? left : each)};
}
// The pages of [from, to) that hold a position of [lo, hi).
__host__ __device__ __forceinline__ void seen_pages(int &from, int &to, int lo, int hi) {
    const int first = lo >> 4, end = (hi >> 4) + ((hi & 15) != 0);
    if (from < first) from = first;
    if (to > end) to = end;
}

// What a workgroup does.
struct Share {
    int kvh;
    int member;     // the group's first row, whose pages are read
    int row0, rows; // the tile's first row and the group's number of rows, (sequence, query head) pairs
    int from, to;   // the split's pages of the prefix
    bool any;       // the workgroup has something to do
};
__device__ __forceinline__ Share share_of(const PrefixParams &p, const Place &w, int tile_rows) {
    Share s;
    // (row tiles in one order / turned, two groups behind up to 8,192 and 4,096 Q8_0 positions: 64 rows at 32/8 heads,
    // d = 128 56.9 / 56.2 us, 40 at 16/8, d = 256 37.3 / 36.0; 64 f32 rows in four at 16/8 111.6 / 113.3)
    const int at = w.x / p.n_kv_heads;  // (the heads run fastest: a head's row tiles share an L2)
    s.kvh = w.x - at * p.n_kv_heads;
    const Tile t = tile_of(p, tile_rows, turned(at, p.columns / p.n_kv_heads, w.y));
    s.any = t.group >= 0;
    if (!s.any) return s;
    const int pages = prefix_positions(p.pre.prefix_len[t.group], p.pre.max_prefix) >> 4;
    s.member = t.first;
    s.rows = t.members * p.group;
    s.row0 = t.at * tile_rows;
    s.from = (w.y + p.pre.first_split) * p.pre.split_pages;
    s.to = min(s.from + p.pre.split_pages, pages);
    s.any = s.from < pages;
    return s;
}

// A lane's row of a tile: the positions it sees and where its query is.
struct Row {
    int lo, hi;  // sees lo <= position < hi
    bool ok;
    int at;  // sequence * n_heads + head (the group's first row, for a row past the group's)
};
__device__ __forceinline__ Row row_of(const PrefixParams &p, const Share &s, int r) {
    Row x;
    x.ok = r < s.rows;
    x.lo = x.hi = 0;
    const int i = x.ok ? r / p.group : 0, b = s.member + i;
    x.at = b * p.n_heads + s.kvh * p.group + (x.ok ? r - i * p.group : 0);
    if (x.ok) {
        const Visible v = visible_of(p.kv_start[b], p.kv_len[b], p.max_kv_len, p.pm.pos_limit, 0);
        x.lo = v.start;
        x.hi = v.n_pages ? v.end : 0;
    }
    return x;
}

// Positions that some row of a wave's tile sees, [wlo, whi), and that all do, [ilo, ihi).
struct Seen {
    int wlo, whi, ilo, ihi;
    __device__ __forceinline__ bool all(int first, int n) const { return first >= ilo && first + n <= ihi; }
};
template <int NT>
__device__ __forceinline__ Seen seen_of(const Row (&rows)[NT]) {
    constexpr int kMost = 0x7fffffff;
    int wlo = kMost, whi = 0, ilo = 0, ihi = kMost;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const Row &r = rows[nt];
        whi = max(whi, (int)wave_extreme<true>((uint32_t)r.hi));
        wlo = min(wlo, (int)wave_extreme<false>((uint32_t)(r.hi > 0 ? r.lo : kMost)));
        ihi = min(ihi, (int)wave_extreme<false>((uint32_t)(r.ok ? r.hi : kMost)));
        ilo = max(ilo, (int)wave_extreme<true>((uint32_t)r.lo));
    }
    return {__builtin_amdgcn_readfirstlane(wlo), __builtin_amdgcn_readfirstlane(whi),
            __builtin_amdgcn_readfirstlane(ilo), __builtin_amdgcn_readfirstlane(ihi)};
}

// A wave's pages again where the rows' windows leave some of the split's unseen; whether they did. A
// page that no row of the tile sees is not read, but for a wave's first, which is asked for before the
// windows are there; a split of which none sees any (`to` <= `from` then) leaves nothing. us a call,
// all pages / these, 32/8 heads, d = 128: 8 rows in windows of 4,096 that begin behind a prefix of
// 32,768 f32 95.7 / 61.2, Q8_0 48 / 35; 16 in 1,024 that begin in 16,384 54 / 45 and 42 / 29.
template <bool EVEN>
__device__ __forceinline__ bool only_seen(Share &s, const Seen &seen, int wave, Pages &mine) {
    const int from = s.from, to = s.to;
    seen_pages(s.from, s.to, seen.wlo, seen.whi);
    if (from == s.from && to == s.to) return false;
    mine = wave_pages<EVEN>(s.from, s.to, wave);
    return true;
}

// Physical pages of a wave's up to 64, one a lane (without any: the sequence's first).
__device__ __forceinline__ int page_ids(const PrefixParams &p, int b, const Pages &w) {
    return (int)map_page(p.pm, b, w.n > 0 ? w.first + min((int)(threadIdx.x & 63), w.n - 1) : 0);
}

// The waves' (m, l) and O, merged and written. A wave's O is in its slot of `slots`
// ([16 NT][D + 4] floats each), scaled to the workgroup's maximum.
constexpr int out_row(int D) { return D + 4; }
template <int D, int NT>
constexpr int kMergeFloats = kWaves * 16 * NT * out_row(D);
// LDS of a workgroup: the queries, later the waves' O; their (m, l); the rows' places; the scales of Q8_0's queries.
template <int D, int NT>
constexpr int kLdsFloats = kMergeFloats<D, NT> + (2 * kWaves + 2) * 16 * NT;

// m of the workgroup for this lane's rows; `put` stores the wave's O, times f[nt], in its slot.
template <int D, int NT, typename Put>
__device__ __forceinline__ void merge_and_store(const PrefixParams &p, const Share &s, int split, float (&m)[NT], float (&l)[NT],
                                                float *slots, float (*mls)[2][16 * NT], const int *at, Put put) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lrow = lane & 15;
    if (lane < 16) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            mls[wave][0][nt * 16 + lrow] = m[nt];
            mls[wave][1][nt * 16 + lrow] = l[nt];
        }
    }
    __syncthreads();  // (and every wave is done with the queries, whose place `slots` takes)
    float f[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float top = mls[0][0][nt * 16 + lrow];
#pragma unroll
        for (int w = 1; w < kWaves; w++) top = fmaxf(top, mls[w][0][nt * 16 + lrow]);
        // (a wave whose scores were all NaN has m = -inf and NaN sums, which stay NaN)
        f[nt] = m[nt] == -INFINITY ? 0.0f : fast_exp2(m[nt] - top);
    }
    put(slots + wave * 16 * NT * out_row(D), f);
    __syncthreads();
    const int64_t first = (int64_t)split * p.n_seqs * p.n_heads;
    for (int i = threadIdx.x; i < 16 * NT * (D / 4); i += kThreads) {
        const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
        if (s.row0 + r >= s.rows) break;
        floatx4 v = *reinterpret_cast<const floatx4 *>(slots + r * out_row(D) + c);
#pragma unroll
        for (int w = 1; w < kWaves; w++)
            v += *reinterpret_cast<const floatx4 *>(slots + (w * 16 * NT + r) * out_row(D) + c);
        *reinterpret_cast<floatx4 *>(p.pre.acc + (first + at[r]) * D + c) = v;
    }
    const int r = threadIdx.x;
    if (r < 16 * NT && s.row0 + r < s.rows) {
        float top = mls[0][0][r], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; w++) top = fmaxf(top, mls[w][0][r]);
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float mw = mls[w][0][r];
            sum = fmaf(mls[w][1][r], mw == -INFINITY ? 0.0f : fast_exp2(mw - top), sum);
        }
        reinterpret_cast<float2 *>(p.pre.ml)[first + at[r]] = make_float2(top, sum);
    }
}

// ---------------------------------------------------------------------------
// f32 storage, on v_mfma_f32_16x16x4_f32: every product and sum is an f32's, so nothing
// is scaled or split. Sums of four products run over the dims kk*16 + kg*4 + j, of lane
// group kg and step j, which makes K and Q four floats of a row a lane, and the d tiles
// of O the dims T*64 + m*4 + c, which makes V so.
// `lds` is kLdsFloats<D, NT> long.
template <int D, int NT, bool CAP>
__device__ __forceinline__ void f32_item(const PrefixParams &p, const Place &w, float *lds) {
    constexpr int KK = D / 16, DT = D / 64;
    static_assert(NT * KK * 256 <= kMergeFloats<D, NT>, "the queries fit where the waves' O will be");
    float(*mls)[2][16 * NT] = reinterpret_cast<float(*)[2][16 * NT]>(lds + kMergeFloats<D, NT>);
    int *row_at = reinterpret_cast<int *>(lds + kMergeFloats<D, NT> + kWaves * 2 * 16 * NT);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lrow = lane & 15, kg = lane >> 4;
    Share sh = share_of(p, w, 16 * NT);
    if (!sh.any) return;

    floatx4 k[KK], v[4][DT];
    const uint32_t koff = (uint32_t)(lrow * p.kv.row_stride + kg * 16);
    const uint32_t voff = (uint32_t)(kg * 4 * p.kv.row_stride + lrow * 16);
    const int64_t head = (int64_t)sh.kvh * p.kv.head_stride;
    const auto load_k = [&](int64_t page) __attribute__((always_inline)) {
        const uint8_t *at = p.kv.k + page * p.kv.page_stride + head;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) k[kk] = *reinterpret_cast<const floatx4 *>(at + koff + kk * 64);
    };
    const auto load_v = [&](int64_t page) __attribute__((always_inline)) {
        const uint8_t *at = p.kv.v + page * p.kv.page_stride + head;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int T = 0; T < DT; T++)
                v[r][T] = *reinterpret_cast<const floatx4 *>(at + voff + r * p.kv.row_stride + T * 256);
    };
    // (the first page is on its way while the queries are; a wave without pages reads the group's first)
    Pages here = wave_pages<false>(sh.from, sh.to, wave);
    int ids = page_ids(p, sh.member, here);
    const auto id = [&](int i) { return (int64_t)__builtin_amdgcn_readlane(ids, min(i, max(here.n, 1) - 1)); };
    load_k(id(0));
    load_v(id(0));

    Row rows[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        rows[nt] = row_of(p, sh, sh.row0 + nt * 16 + lrow);
        if (threadIdx.x < 16) row_at[nt * 16 + lrow] = rows[nt].at;
    }
    // the queries, [nt][kk][lane] in the order in which a lane reads them: a wave takes every fourth kk
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int k4 = 0; k4 < KK / kWaves; k4++) {
            const int kk = k4 * kWaves + wave;
            floatx4 x = *reinterpret_cast<const floatx4 *>(p.q + (int64_t)rows[nt].at * D + kk * 16 + kg * 4) * p.q_mul;
            if (!rows[nt].ok) x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            reinterpret_cast<floatx4 *>(lds)[(nt * KK + kk) * 64 + lane] = x;
        }
    const Seen seen = seen_of<NT>(rows);
    if (only_seen<false>(sh, seen, wave, here)) {
        if (sh.from >= sh.to) return;  // (all waves: they have the same rows)
        ids = page_ids(p, sh.member, here);
        load_k(id(0));
        load_v(id(0));
    }
    const int n = here.n;
    __syncthreads();
    const floatx4 *qs = reinterpret_cast<const floatx4 *>(lds);

    floatx4 o[DT][4][NT];  // O of d = T*64 + (kg*4 + r)*4 + c in [T][c][nt][r]
    float m[NT], lpart[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt] = -INFINITY;
        lpart[nt] = 0.0f;
#pragma unroll
        for (int T = 0; T < DT; T++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[T][c][nt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    {
        for (int i = 0; i < n; i++) {
            const int first = (here.first + i) * 16;
            const bool inside = seen.all(first, 16);
            int qi = lane;
            asm volatile("" : "+v"(qi));  // (read anew for every page: kept, they would crowd the other registers)
            floatx4 s[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[nt][0] = s[nt][1] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                floatx4 q[NT];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) q[nt] = qs[qi + (nt * KK + kk) * 64];
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
                        s[nt][j & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[kk][j], q[nt][j], s[nt][j & 1], 0, 0, 0);
            }
            load_k(id(i + 1));
            float pr[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                floatx4 x = s[nt][0] + s[nt][1];
                if constexpr (CAP) {
                    const SoftCap f(p.softcap);
#pragma unroll
                    for (int r = 0; r < 4; r++) x[r] = f(x[r]);
                }
                if (!inside) {
                    const int pos0 = rare(first + kg * 4);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int pos = pos0 + r;
                        x[r] = pos >= rows[nt].lo && pos < rows[nt].hi ? x[r] : -INFINITY;
                    }
                }
                const float mine = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                if (__ballot(mine > m[nt] + kLazy)) {
                    const float f = moved(m[nt], mine, kLazy);
                    lpart[nt] *= f;
#pragma unroll
                    for (int T = 0; T < DT; T++)
#pragma unroll
                        for (int c = 0; c < 4; c++) o[T][c][nt] *= f;
                }
                const float off = m[nt] == -INFINITY ? 0.0f : m[nt];
#pragma unroll
                for (int r = 0; r < 4; r++) pr[nt][r] = fast_exp2(x[r] - off);
                lpart[nt] += (pr[nt][0] + pr[nt][1]) + (pr[nt][2] + pr[nt][3]);
            }
            // A value that is infinite or NaN reaches only the rows that see its position (0 times
            // it would not be 0): where some row does not, and there is one, those are left out
            // of the product and added by themselves.
            bool apart = false;
            if (!inside) {
                float z = rare(0.0f);
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int T = 0; T < DT; T++)
#pragma unroll
                        for (int c = 0; c < 4; c++) z = fmaf(v[r][T][c], 0.0f, z);
                apart = __ballot(z != z) != 0;
                if (apart) {
                    const float inf = rare(INFINITY);
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int T = 0; T < DT; T++)
#pragma unroll
                            for (int c = 0; c < 4; c++) v[r][T][c] = fabsf(v[r][T][c]) < inf ? v[r][T][c] : 0.0f;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int T = 0; T < DT; T++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            o[T][c][nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][T][c], pr[nt][r], o[T][c][nt], 0, 0, 0);
            if (apart) {
                const uint8_t *at = p.kv.v + id(i) * p.kv.page_stride + head + kg * 64;
#pragma unroll 1
                for (int k4 = 0; k4 < 4; k4++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int key = 4 * k4 + j, pos = first + key;
                        float pk[NT];
                        bool sees[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            pk[nt] = __shfl(pr[nt][j], k4 * 16 + lrow);
                            sees[nt] = pos >= rows[nt].lo && pos < rows[nt].hi;
                        }
#pragma unroll
                        for (int T = 0; T < DT; T++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const floatx4 w =
                                    *reinterpret_cast<const floatx4 *>(at + key * p.kv.row_stride + T * 256 + r * 16);
#pragma unroll
                                for (int c = 0; c < 4; c++)
#pragma unroll
                                    for (int nt = 0; nt < NT; nt++) {
                                        const float x = o[T][c][nt][r];
                                        o[T][c][nt][r] = sees[nt] && !(fabsf(w[c]) < INFINITY) ? fmaf(pk[nt], w[c], x) : x;
                                    }
                                asm volatile("" ::: "memory");  // (one row of values at a time in registers)
                            }
                    }
                }
            }
            load_v(id(i + 1));
        }
    }
    float l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) l[nt] = sum_rows4(lpart[nt]);
    merge_and_store<D, NT>(p, sh, w.y, m, l, lds, mls, row_at, [&](float *slot, const float (&f)[NT]) __attribute__((always_inline)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int T = 0; T < DT; T++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const floatx4 x = {o[T][0][nt][r], o[T][1][nt][r], o[T][2][nt][r], o[T][3][nt][r]};
                    *reinterpret_cast<floatx4 *>(slot + (nt * 16 + lrow) * out_row(D) + T * 64 + kg * 16 + r * 4) = x * f[nt];
                }
    });
}

// ---------------------------------------------------------------------------
// Q8_0 storage, on v_mfma_f32_16x16x32_f16, as the decode of single rows has it
// (gla_decode_q8.hip): quants are exact in f16; queries, and probabilities times the
// values' scales, are two f16 pieces (hi = f16(x), lo = f16(x - hi)) after a power-of-two
// rescale that puts the largest below 2^14. A step is two pages, the depth of one product
// with V; K's scales are applied to the scores of each block.

// Four stored quants (x + 128, in byte order) -> halves at..at+3 of `o`: 0x64XX is
// 1024 + XX in f16, so subtracting 1152 leaves x exactly.
__device__ __forceinline__ void quants4(uint32_t u, half8 &o, int at) {
    const half2v bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    const half2v a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
    const half2v c = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
    o[at + 0] = a[0];
    o[at + 1] = a[1];
    o[at + 2] = c[0];
    o[at + 3] = c[1];
}
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) {
    return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w));
}
template <int N>
__device__ __forceinline__ float half_at(const uint32_t (&a)[N], int i) {
    const uint32_t w = a[i >> 1];
    return (float)__builtin_bit_cast(_Float16, (uint16_t)((i & 1) ? (w >> 16) : (w & 0xffff)));
}
// e with x = m * 2^e, m in [0.5, 1); scaling by 2^(14 - e) maps max|.| below 2^14.
__device__ __forceinline__ int pow2_exp(float x) {
    int e = 0;
    (void)frexpf(x, &e);
    return e < -100 ? -100 : (e > 100 ? 100 : e);
}
template <int N>
__device__ __forceinline__ void load_words(const uint8_t *src, uint32_t (&dst)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 w = reinterpret_cast<const uint4 *>(src)[i];
            dst[4 * i] = w.x;
            dst[4 * i + 1] = w.y;
            dst[4 * i + 2] = w.z;
            dst[4 * i + 3] = w.w;
        }
    } else {
        static_assert(N == 2, "8 bytes");
        const uint2 w = *reinterpret_cast<const uint2 *>(src);
        dst[0] = w.x;
        dst[1] = w.y;
    }
}

// The f16 pieces of p[j] * scale[j], hi = f16(p * scale) and lo = f16(p * scale - hi), of the
// f16 scales in the words' high (HIGH) or low halves: written so that products and remainders
// become mixed multiply-adds, which take the halves as they are. 24 instructions where assembly
// needs 16, but the compiler counts the wait states between the matrix instructions and the
// registers that these write. Assembly would have to wait for the longest of them every time,
// which is no faster: 64 rows of 64-1,000 positions behind 8,192 at 32/8 heads, d = 128 53.0 us
// / this 51.2, of 8-64 47.4 / 45.9, 96 rows in 3 groups 84.0 / 81.8, d = 256 58.5 / 57.9.
template <bool HIGH>
__device__ __forceinline__ void pieces8(const float (&p)[8], const uint32_t (&w)[8], half8 &hi, half8 &lo) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float s0 = half_at(w, 2 * j + HIGH), s1 = half_at(w, 2 * j + 2 + HIGH);
        const half2v h = __builtin_convertvector((float2v){fmaf(p[j], s0, 0.0f), fmaf(p[j + 1], s1, 0.0f)}, half2v);
        hi[j] = h[0];
        hi[j + 1] = h[1];
        lo[j] = (_Float16)fmaf(p[j], s0, -(float)h[0]);
        lo[j + 1] = (_Float16)fmaf(p[j + 1], s1, -(float)h[1]);
    }
}

template <int D, int NT, bool CAP>
__device__ __forceinline__ void q8_item(const PrefixParams &p, const Place &w, float *lds) {
    constexpr int NB = D / 32, NQ = D / 64, ND = D / 16;
    static_assert(NT * NB * 2 * 256 <= kMergeFloats<D, NT>, "the queries' pieces fit where the waves' O will be");
    float(*mls)[2][16 * NT] = reinterpret_cast<float(*)[2][16 * NT]>(lds + kMergeFloats<D, NT>);
    int *row_at = reinterpret_cast<int *>(lds + kMergeFloats<D, NT> + kWaves * 2 * 16 * NT), *qexp = row_at + 16 * NT;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lrow = lane & 15, kg = lane >> 4;
    Share sh = share_of(p, w, 16 * NT);
    if (!sh.any) return;

    const uint8_t *base = p.kv.k + (int64_t)sh.kvh * p.kv.head_stride;
    uint4 k[2][NQ], v[2][NQ];
    uint32_t ks[2][2][NB], vs[2][2 * NB];  // 4 positions x the blocks of a parity; x all blocks
    const uint32_t off = lane * 16, ksoff = (uint32_t)(32 * D + kg * 4 * NB), vsoff = (uint32_t)(33 * D + kg * 8 * NB);
    const auto load_k = [&](int P, int64_t page) __attribute__((always_inline)) {
        const uint8_t *at = base + page * p.kv.page_stride;
#pragma unroll
        for (int c = 0; c < NQ; c++) k[P][c] = *reinterpret_cast<const uint4 *>(at + off + c * 1024);
        load_words(at + ksoff, ks[P][0]);
        load_words(at + ksoff + 16 * NB, ks[P][1]);
    };
    const auto load_v = [&](int P, int64_t page) __attribute__((always_inline)) {
        const uint8_t *at = base + page * p.kv.page_stride;
#pragma unroll
        for (int c = 0; c < NQ; c++) v[P][c] = *reinterpret_cast<const uint4 *>(at + 16 * D + off + c * 1024);
        load_words(at + vsoff, vs[P]);
    };
    // (the first pages are on their way while the queries are split; a wave without pages reads the group's first)
    Pages here = wave_pages<true>(sh.from, sh.to, wave);
    int ids = page_ids(p, sh.member, here);
    const auto id = [&](int i) { return (int64_t)__builtin_amdgcn_readlane(ids, min(i, max(here.n, 1) - 1)); };
    const auto load_first = [&]() __attribute__((always_inline)) {
        load_k(0, id(0));
        load_k(1, id(1));
        load_v(0, id(0));
        load_v(1, id(1));
    };
    load_first();

    Row rows[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        rows[nt] = row_of(p, sh, sh.row0 + nt * 16 + lrow);
        if (threadIdx.x < 16) row_at[nt * 16 + lrow] = rows[nt].at;
    }
    // the queries' pieces, [nt][block][piece][lane]: wave w takes the tiles nt = w, w + 4, ...
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        if (nt % kWaves != wave) continue;
        const float *qp = p.q + (int64_t)rows[nt].at * D + kg * 8;
        float x[NB][8], top = 0.0f;
#pragma unroll
        for (int blk = 0; blk < NB; blk++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const floatx4 w = *reinterpret_cast<const floatx4 *>(qp + blk * 32 + h * 4) * p.q_mul;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[blk][4 * h + e] = w[e];
                    top = fmaxf(top, fabsf(w[e]));
                }
            }
        // an infinite entry's second piece is 0 and its score infinite; the scale is the finite entries'
        const bool infinite = __ballot(top == INFINITY) != 0;
        if (infinite) {
            top = rare(0.0f);
#pragma unroll
            for (int blk = 0; blk < NB; blk++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float a = fabsf(x[blk][j]);
                    top = a < INFINITY ? fmaxf(top, a) : top;
                }
        }
        top = max_rows4(top);
        const int e = pow2_exp(top);
        const float mul = rows[nt].ok ? ldexpf(1.0f, 14 - e) : 0.0f;
        if (kg == 0) qexp[nt * 16 + lrow] = e;
#pragma unroll
        for (int blk = 0; blk < NB; blk++) {
            half8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = x[blk][j] * mul;
                hi[j] = (_Float16)y;
                lo[j] = (_Float16)(y - (float)hi[j]);
            }
            if (infinite) {
                const float inf = rare(INFINITY);
#pragma unroll
                for (int j = 0; j < 8; j++) lo[j] = fabsf(x[blk][j]) == inf ? (_Float16)0.0f : lo[j];
            }
            half8 *to = reinterpret_cast<half8 *>(lds) + (nt * NB + blk) * 2 * 64 + lane;
            to[0] = hi;
            to[64] = lo;
        }
    }
    const Seen seen = seen_of<NT>(rows);
    if (only_seen<true>(sh, seen, wave, here)) {
        if (sh.from >= sh.to) return;  // (all waves: they have the same rows)
        ids = page_ids(p, sh.member, here);
        load_first();
    }
    const int n = here.n;
    __syncthreads();
    const half8 *qs = reinterpret_cast<const half8 *>(lds);
    float sm[NT];  // undoes a query's scale
#pragma unroll
    for (int nt = 0; nt < NT; nt++) sm[nt] = ldexpf(1.0f, qexp[nt * 16 + lrow] - 14);

    floatx4 o[ND][NT];  // O of d = t*16 + kg*4 + r
    float m[NT], moff[NT], lpart[NT];  // p 2^vexp = 2^(s + moff)
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt] = -INFINITY;
        moff[nt] = lpart[nt] = 0.0f;
#pragma unroll
        for (int t = 0; t < ND; t++) o[t][nt] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // O and the sums of P are in units of 2^-vexp. Where m's own unit is so large that vexp - m would be
    // rounded to it (an m that keeps p below 2^2 all the same), in units of 1: products of f16 scales fit.
    int vexp = 0;
    const auto exp_of = [&](float m) { return fabsf(m) < 0x1p22f ? vexp : min(vexp, 0); };
    if (n > 0) {
        // P' = p * vscale * 2^vexp is below 2^14 for p = 1
        const int units = n * (D / 16);  // 16 bytes of V scales each
        const auto largest = [&](auto finite) {
            float top = 0.0f;
            for (int u0 = 0; u0 < units; u0 += 64) {
                const int u = min(u0 + lane, units - 1);
                const int64_t page = __shfl(ids, u / (D / 16));
                uint32_t w[4];
                load_words(base + page * p.kv.page_stride + 33 * D + u % (D / 16) * 16, w);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x = fabsf(half_at(w, i));
                    top = finite && x == INFINITY ? top : fmaxf(top, x);
                }
            }
            return wave_max(top);
        };
        float vmax = largest(std::false_type{});
        // (an infinite scale has no power of two: it is the finite ones', whose positions some rows may see alone)
        const bool vinf = __ballot(vmax == INFINITY) != 0;
        if (vinf) vmax = largest(std::true_type{});
        const int ve = __builtin_amdgcn_readfirstlane(pow2_exp(vmax));
        vexp = 14 - ve;

        for (int i = 0; i < n; i += 2) {
            const int first = (here.first + i) * 16;
            const bool two = i + 1 < n;
            const bool plain = two && !vinf && seen.all(first, 32);  // every row sees all, and no scale is infinite
            int qi = lane;
            asm volatile("" : "+v"(qi));  // (read anew for every step: kept, they would crowd the other registers)
            floatx4 s[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[nt][0] = s[nt][1] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int blk = 0; blk < NB; blk++) {
                half8 a[2];
#pragma unroll
                for (int P = 0; P < 2; P++) {
                    quants4(word(k[P][blk >> 1], (blk & 1) * 2), a[P], 0);
                    quants4(word(k[P][blk >> 1], (blk & 1) * 2 + 1), a[P], 4);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const half8 qh = qs[qi + (nt * NB + blk) * 128], ql = qs[qi + (nt * NB + blk) * 128 + 64];
                    floatx4 t[2];
#pragma unroll
                    for (int P = 0; P < 2; P++)
                        t[P] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[P], qh, floatx4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                    for (int P = 0; P < 2; P++) t[P] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[P], ql, t[P], 0, 0, 0);
#pragma unroll
                    for (int P = 0; P < 2; P++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            s[nt][P][r] = fmaf(half_at(ks[P][blk & 1], r * (NB / 2) + (blk >> 1)), t[P][r], s[nt][P][r]);
                }
            }
            load_k(0, id(i + 2));
            load_k(1, id(i + 3));

            float pr[NT][8];
            uint32_t sees[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                floatx4 x[2] = {s[nt][0], s[nt][1]};
                if constexpr (CAP) {
                    x[0] *= sm[nt];
                    x[1] *= sm[nt];
                    const SoftCap f(p.softcap);
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j >> 2][j & 3] = f(x[j >> 2][j & 3]);
                }
                sees[nt] = 0xff;
                if (!plain) {
                    const int pos0 = rare(first + kg * 4);
                    sees[nt] = 0;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int pos = pos0 + (j >> 2) * 16 + (j & 3);
                        const bool ok = pos >= rows[nt].lo && pos < rows[nt].hi && (j < 4 || two);
                        sees[nt] |= ok ? 1u << j : 0u;
                        x[j >> 2][j & 3] = ok ? x[j >> 2][j & 3] : -INFINITY;
                    }
                }
                const float c = CAP ? 1.0f : sm[nt];
                const float mine = c * fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                                             fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
                if (__ballot(mine > m[nt] + kLazyQ8)) {
                    const int was = exp_of(m[nt]);
                    const float f = ldexpf(moved(m[nt], mine, kLazyQ8), exp_of(m[nt]) - was);
                    moff[nt] = m[nt] == -INFINITY ? 0.0f : (float)exp_of(m[nt]) - m[nt];
                    lpart[nt] *= f;
#pragma unroll
                    for (int t = 0; t < ND; t++) o[t][nt] *= f;
                }
#pragma unroll
                for (int j = 0; j < 8; j++) pr[nt][j] = fast_exp2(fmaf(x[j >> 2][j & 3], c, moff[nt]));
                lpart[nt] += ((pr[nt][0] + pr[nt][1]) + (pr[nt][2] + pr[nt][3])) +
                             ((pr[nt][4] + pr[nt][5]) + (pr[nt][6] + pr[nt][7]));
            }

#pragma unroll
            for (int blk = 0; blk < NB; blk++) {
                half8 a[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int t = 2 * blk + h;
                    quants4(word(v[0][t >> 2], t & 3), a[h], 0);
                    quants4(word(v[1][t >> 2], t & 3), a[h], 4);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    half8 hi, lo;
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) w[j] = vs[j >> 2][((j & 3) * NB + blk) >> 1];
                    if (blk & 1)
                        pieces8<true>(pr[nt], w, hi, lo);
                    else
                        pieces8<false>(pr[nt], w, hi, lo);
                    // a scale that is infinite or NaN, at a position that the row does not see
                    // (nothing) or sees (infinity has no second piece)
                    if (!plain) {
                        const uint32_t has = rare(sees[nt]);
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            lo[j] = (has >> j & 1) == 0 || __builtin_isinf((float)hi[j]) ? (_Float16)0.0f : lo[j];
                            hi[j] = has >> j & 1 ? hi[j] : (_Float16)0.0f;
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        o[2 * blk + h][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[h], hi, o[2 * blk + h][nt], 0, 0, 0);
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        o[2 * blk + h][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[h], lo, o[2 * blk + h][nt], 0, 0, 0);
                }
            }
            load_v(0, id(i + 2));
            load_v(1, id(i + 3));
        }
    }
    float l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) l[nt] = ldexpf(sum_rows4(lpart[nt]), -exp_of(m[nt]));
    merge_and_store<D, NT>(p, sh, w.y, m, l, lds, mls, row_at, [&](float *slot, const float (&f)[NT]) __attribute__((always_inline)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int t = 0; t < ND; t++)
                *reinterpret_cast<floatx4 *>(slot + (nt * 16 + lrow) * out_row(D) + t * 16 + kg * 4) =
                    o[t][nt] * ldexpf(f[nt], -exp_of(m[nt]));
    });
}

// The one launch of a batch behind its prefixes: the prefixes' workgroups, then, where those
// leave room, those of the rows' own pages. us a call, in two launches / in one / in one with both
// kinds in turn: Q8_0 behind 8,192 positions at 32/8 heads, d = 128, 64 rows of 64-1,000 64.0 /
// 60.3 / 73.2, of 8-64 53.3 / 52.1 / 61.9, 4 rows 24.3 / 18.6 / 20.0; 64 rows in 4 groups behind
// 2,048 35.3 / 28.1 / 35.9 (the prefixes' are the longest, and all of them are resident).
struct Mixed {
    int px, py, n_prefix;  // the prefixes' columns and splits, and their product
    int ox, oy, n_own;     // those of the rows' own pages
    // (the rows' begin on the same XCD as in a launch of their own)
    __host__ __device__ int own0() const { return (n_prefix + 7) & ~7; }
    // True for a workgroup of the prefixes, at `w`, false for one of the rows' (w.z < 0: none of either).
    __device__ __forceinline__ bool place(Place &w) const {
        int i = (int)(blockIdx.y * gridDim.x + blockIdx.x);
        const bool of_prefix = i < own0();
        if (!of_prefix) i -= own0();
        const int nx = of_prefix ? px : ox, ny = of_prefix ? py : oy;
        const int row = i / nx;
        w.x = i - row * nx;
        w.z = row / ny;
        w.y = row - w.z * ny;
        if (i >= (of_prefix ? n_prefix : n_own)) w.z = -1;
        return of_prefix;
    }
    // (a grid's row holds fewer than 2^32 threads)
    dim3 grid() const {
        const unsigned n = (unsigned)(own0() + n_own), most = 1u << 23;
        return dim3(n < most ? n : most, (n - 1) / most + 1);
    }
};

}  // namespace prefix
}  // namespace gla
