// gla_decode_prefix.hip -- when and in how many splits a batch's shared prefixes are read
// apart (host code; the kernels' part is gla_prefix.h).
#include <stdlib.h>

#include <algorithm>
#include <vector>

#include "gla_prefix.h"

namespace gla {

namespace {
struct Pages {
    int from, to;
};
// What a launch's rows attend, in positions: exactly, from host copies, or as far as its bounds say.
struct Work {
    int64_t saved = 0;  // that they would read again, row by row
    int64_t own = 0;    // behind their prefixes, or in none
    int64_t total = 0;
    int longest = 0;    // of a prefix that several rows share, what some row sees
};
}  // namespace

// Whether reading the prefixes apart is the faster way. It costs
// a combine and the set-up of more workgroups; what it saves are the bytes that the rows
// would read again (from L2 mostly) and, with Q8_0, the length of a wave's chain of pages.
// us a call, apart / row by row, in a captured step with 1-33 positions of each row's own:
//   f32   9/3 heads, d = 64:   8 rows of 2,048 (22 MB saved) 12.6 / 10.8, 8 of 4,096 (44 MB) 13.7 / 13.8, 16 of 4,096 14.8 / 20.2
//        32/8 heads, d = 128:  8 rows of 256 (15 MB) 15.8 / 11.4, 16 of 256 (31 MB) 16.5 / 16.8, 4 of 2,048 (50 MB) 14.9 / 22.5
//        16/8 heads, d = 256:  4 rows of 704 (35 MB) 19.1 / 14.9, 16 of 256 (63 MB) 18.9 / 17.7, 8 of 704 (81 MB) 20.1 / 22.2
//   Q8_0  9/3 heads, d = 64:   2 rows of 256 9.9 / 8.1, of 704 10.3 / 10.8, of 4,096 14.4 / 20.9, 16 of 704 11.1 / 11.8
//        32/8 heads, d = 128:  2 rows of 256 10.8 / 9.6, of 704 11.0 / 13.6, 16 of 256 12.8 / 12.9
//        16/8 heads, d = 256:  2 rows of 256 13.2 / 13.6, 8 of 256 13.9 / 13.8, 2 of 704 13.4 / 19.9
// It also costs where rows have much of their own, or share nothing: f32 at head_dim 256 reads a row's
// own positions once a head (a wave holds one, so those of a KV head's others are read again), other
// f32 kernels lose their merge, and Q8_0 takes rows of no group through the prefixes' tiles. A pair that
// shares 512 positions among 64 rows of 2,000 f32 at 16/8, d = 256 594 / 373 us, at 32/8, d = 128 254 /
// 238, Q8_0 52 / 52; 16 rows that see 1,050 of a prefix and 1,000 of their own f32 at 16/8 84 / 78; 64
// lone rows behind 1,024 beside a pair behind 64 Q8_0 at 32/8 36 / 31, 16 behind 2,048 beside a pair
// behind as many at 16/8 46 / 75 (5% saved).
static bool pays(const DecodeLaunch &d, const Work &w) {
    const int64_t position = d.kv.page_stride / 16;  // bytes
    if (w.longest == 0) return false;
    if (const char *env = getenv("GLA_DECODE_PREFIX")) return atoi(env) != 0;  // (tuning and tests)
    if (d.q8) return w.longest >= (d.head_dim == 64 ? 640 : 448) && 64 * w.saved >= w.total;
    const bool wide = d.head_dim == 256;
    const int64_t own = wide && d.n_heads > d.n_kv_heads ? w.own : w.own / 10;
    return (w.saved - own) * position >= (wide ? 70000000 : 30000000);
}

void plan_prefix(const gla_ctx *ctx, DecodeLaunch *launch) {
    const DecodeLaunch &d = *launch;
    PrefixLaunch *pre = &launch->pre;
    const bool host = pre->group_start_host != nullptr;
    // The bounds, as near as the host copies let them be, and the pages of each group's prefix that some row sees.
    std::vector<Pages> seen;
    Work work;
    if (host) {
        seen.resize(pre->n_groups);
        int max_group = 0, max_prefix = 0;
        for (int g = 0; g < pre->n_groups; g++) {
            const int first = pre->group_start_host[g], end = pre->group_start_host[g + 1];
            const int positions = prefix_positions(pre->prefix_len_host[g], pre->max_prefix);
            max_group = std::max(max_group, end - first);
            max_prefix = std::max(max_prefix, positions);
            int lo = positions, hi = 0, n = 0;
            int64_t all = 0;
            for (int b = first; b < end; b++) {
                if (d.kv_len_host[b] == 0 || d.kv_start_host[b] >= positions) continue;
                const int to = std::min(positions, d.kv_start_host[b] + d.kv_len_host[b]);
                lo = std::min(lo, (int)d.kv_start_host[b]);
                hi = std::max(hi, to);
                all += to - d.kv_start_host[b];
                n++;
            }
            seen[g] = {lo / 16, (hi + 15) / 16};
            if (n > 1) {
                work.saved += std::max<int64_t>(all - (hi - lo), 0);
                work.longest = std::max(work.longest, hi - lo);
                work.own -= all;
            }
        }
        for (int b = 0; b < d.n_seqs; b++) work.total += d.kv_len_host[b];
        work.own += work.total;
        pre->max_group = max_group;
        pre->max_prefix = max_prefix;
    } else if (pre->max_group > 1) {
        // (what the rows of groups have of their own is between nothing and the bound of every replay: it is
        // left out, so that it does not hide what they share)
        const int64_t most = std::min<int64_t>(d.n_seqs, (int64_t)pre->n_groups * pre->max_group);
        work.longest = std::min(pre->max_prefix, d.max_kv_len);
        work.saved = std::min<int64_t>(d.n_seqs - pre->n_groups, (int64_t)pre->n_groups * (pre->max_group - 1)) * work.longest;
        work.own = (d.n_seqs - most) * std::min(pre->max_own, d.max_kv_len);
        work.total = work.own + most * work.longest;
    }
    if (!pays(d, work)) {
        pre->n_groups = 0;
        return;
    }
    const int64_t tile = 16 * prefix_tiles(d), group = d.n_heads / d.n_kv_heads;
    const int pages = pre->max_prefix / 16;
    int64_t tiles = 0;
    for (int g = 0; host && g < pre->n_groups; g++)
        tiles += ((pre->group_start_host[g + 1] - pre->group_start_host[g]) * group + tile - 1) / tile;
    if (!host)
        tiles = std::min<int64_t>(pre->n_groups * ((pre->max_group * group - 1) / tile + 1), d.n_seqs * group / tile + pre->n_groups);
    // The launch has a workgroup for each of these a split, and those find their group: one for every
    // tile of the largest group a group are thousands too many where groups are unlike. 64 rows behind
    // 2,048 and 63 pairs behind 64-1,924 at 32/8 heads, d = 128, such / these: f32 365 / 173 us, Q8_0
    // 146 / 71 (row by row 469 and 80); 8 groups of 1-32 rows behind 100-8,192 known by their bounds alone
    // 284 / 154 and 109 / 74; 3 of 96 Q8_0 rows behind 8,192 85 / 82.
    pre->tiles = (int)std::min<int64_t>(tiles, 1 << 30);  // (as many are refused with the grid)
    // workgroups of a launch with splits of n pages: as they are, or from the bounds
    const bool few = host && pre->n_groups <= 256;
    const auto wgs = [&](int n) {
        int64_t sum = 0;
        for (int g = 0; few && g < pre->n_groups; g++) {
            const int64_t rows = (pre->group_start_host[g + 1] - pre->group_start_host[g]) * group;
            if (seen[g].from < seen[g].to) sum += (rows + tile - 1) / tile * ((seen[g].to - 1) / n - seen[g].from / n + 1);
        }
        return (few ? sum : tiles * ((pages + n - 1) / n)) * d.n_kv_heads;
    };
    // the fewest pages (a wave's: an even number, at most 64) that leave at most `most` workgroups
    const auto pages_for = [&](int64_t most) {
        int lo = 1, hi = 32;  // (eights; more pages never make more workgroups)
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (wgs(8 * mid) > most)
                lo = mid + 1;
            else
                hi = mid;
        }
        return 8 * lo;
    };
    // A workgroup for every unit, which leaves room on each for the rows' own: with more the waves'
    // set-up and the combine's splits cost more than they give. Half as many more for several
    // groups, whose unlike lengths and part-filled tiles leave units idle. us a call, 1 / 1.5 / 2 a
    // unit: behind 8,192 positions at 32/8 heads, d = 128, 64 rows of 64-1,000 Q8_0 54.6 / 61 (2), of
    // 8-64 f32 102 / 109 (2); in groups 96 Q8_0 rows in 3 93 / 88 / 88, 48 f32 rows in 3 133 / 95 / 94,
    // 64 Q8_0 rows in 4 behind 2,048 32.9 / 27.6 / 29.5; at 16/8, d = 256 24 f32 rows in 3 behind up to
    // 4,096 64.5 / 63.1 / 67.6, 40 Q8_0 rows in 2 34.8 / 39.0 / 42.0.
    // Three a unit for several groups known by their bounds alone, of which most may be shorter: 8 Q8_0
    // groups of 1-32 rows behind 100-8,192, the longest one row's (35 us row by row), 1.5 / 3 / 6 a unit
    // 74 / 46 / 37, f32 154 / 97 / 77, with the host copies 36 and 65; 32 pairs behind 2,048 each Q8_0 33 /
    // 37 / 42, f32 109 / 116 / 121.
    const int units = ctx->n_cu;
    pre->split_pages = pages_for(pre->n_groups <= 1 ? units : (few ? units + units / 2 : 3 * units));
    int from = pages, to = 0;
    for (const Pages &p : seen)
        if (p.from < p.to) from = std::min(from, p.from), to = std::max(to, p.to);
    if (!host) from = 0, to = pages;
    pre->first_split = to > from ? from / pre->split_pages : 0;
    pre->n_splits = to > from ? (to - 1) / pre->split_pages - pre->first_split + 1 : 0;
}

void prefix_params(const DecodeLaunch &d, void *scratch, PrefixLaunch *out, prefix::PrefixParams *prm) {
    *out = d.pre;
    out->acc = (float *)scratch;
    out->ml = out->acc + (size_t)d.pre.n_splits * d.n_seqs * d.n_heads * d.head_dim;
    prm->kv = d.kv;
    prm->pm = d.pm;
    prm->pre = *out;
    prm->q = d.q;
    prm->kv_start = d.kv_start;
    prm->kv_len = d.kv_len;
    prm->max_kv_len = d.max_kv_len;
    prm->n_seqs = d.n_seqs;
    prm->n_heads = d.n_heads;
    prm->n_kv_heads = d.n_kv_heads;
    prm->group = d.n_heads / d.n_kv_heads;
    const bool cap = d.softcap > 0.0f;
    prm->q_mul = cap ? d.scale : d.scale * lanes::kLog2e;
    prm->softcap = cap ? d.softcap : 0.0f;
    // (more than 2^30 are refused with the grid)
    prm->columns = (int)std::min<int64_t>((int64_t)d.pre.tiles * d.n_kv_heads, 1 << 30);
}

int mix_prefix(const DecodeLaunch &d, const prefix::PrefixParams &prm, dim3 own, prefix::Mixed *mix) {
    const int64_t n_prefix = (int64_t)prm.columns * d.pre.n_splits, n_own = (int64_t)own.x * own.y * own.z;
    if (n_prefix > 1 << 30 || n_own > (1 << 30) - 8)
        return set_error(GLA_ERR_INVALID, "decode: %lld workgroups for shared prefixes and %lld for the rows behind them",
                         (long long)n_prefix, (long long)n_own);
    *mix = {prm.columns, d.pre.n_splits, (int)n_prefix, (int)own.x, (int)own.y, (int)n_own};
    return GLA_OK;
}

}  // namespace gla
