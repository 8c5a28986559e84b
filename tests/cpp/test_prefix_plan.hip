// How gla_decode_shared plans a batch's prefixes (plan_prefix, mix_prefix) and which pages a wave of them reads, on the
// host, without a device.
#include <stdarg.h>
#include <stdio.h>

#include <set>
#include <vector>

#include "../../glint_amd/csrc/gla_decode_prefix.hip"

namespace gla {
int set_error(int code, const char *, ...) { return code; }
}  // namespace gla

namespace {

using namespace gla;

#define CHECK(cond, ...)                         \
    do {                                         \
        if (!(cond)) {                           \
            printf("%s: ", #cond), printf(__VA_ARGS__); \
            printf("\n");                        \
            return 1;                            \
        }                                        \
    } while (0)

struct Shape {
    int heads, kv_heads, d;
};
constexpr Shape kShapes[] = {{9, 3, 64}, {32, 8, 128}, {16, 8, 256}};

struct Batch {
    std::vector<int32_t> starts, prefix, start, len;  // groups; windows of the rows
    DecodeLaunch d{};
    Batch(const Shape &s, bool q8, const std::vector<int> &sizes, std::vector<int32_t> lens, int own, bool host, int window = 0,
          int more = 0)
        : starts{0}, prefix(lens) {
        for (int n : sizes) starts.push_back(starts.back() + n);
        const int n = starts.back() + more;
        for (int b = 0, g = 0; b < n; b++) {
            while (g < (int)sizes.size() && starts[g + 1] <= b) g++;
            const int end = (g < (int)sizes.size() ? prefix[g] : 0) + own;
            start.push_back(window && end > window ? end - window : 0);
            len.push_back(end - start.back());
        }
        d.q8 = q8;
        d.head_dim = s.d;
        d.n_heads = s.heads;
        d.n_kv_heads = s.kv_heads;
        d.n_seqs = n;
        d.pm.pos_limit = 1 << 20;
        const int64_t row = (int64_t)s.kv_heads * s.d;
        d.kv.page_stride = 16 * (q8 ? row * 2 * 34 / 32 : row * 8);
        d.max_kv_len = *std::max_element(len.begin(), len.end());
        d.pre.n_groups = (int)sizes.size();
        d.pre.max_group = *std::max_element(sizes.begin(), sizes.end());
        d.pre.max_prefix = *std::max_element(lens.begin(), lens.end()) & ~15;
        d.pre.max_own = own;
        if (host) {
            d.kv_start_host = start.data();
            d.kv_len_host = len.data();
            d.pre.group_start_host = starts.data();
            d.pre.prefix_len_host = prefix.data();
        }
    }
    void plan() {
        gla_ctx ctx{};
        ctx.n_cu = 256;
        plan_prefix(&ctx, &d);
    }
};

// Every row tile of a batch has a workgroup in each split, and a launch that knows its groups has no others.
int tiles() {
    for (const Shape &s : kShapes)
        for (bool q8 : {false, true})
            for (bool host : {false, true})
                for (const auto &sizes : {std::vector<int>{64}, {64, 2, 2, 2, 2, 2, 2, 2, 2}, std::vector<int>(300, 2), {1, 1, 40, 3, 0, 7}}) {
                    std::vector<int32_t> lens(sizes.size(), 4096);
                    Batch b(s, q8, sizes, lens, 20, host);
                    b.plan();
                    CHECK(b.d.pre.n_groups == (int)sizes.size(), "%d groups of %d/%d heads", (int)sizes.size(), s.heads, s.kv_heads);
                    prefix::PrefixParams prm{};
                    PrefixLaunch placed;
                    prefix_params(b.d, nullptr, &placed, &prm);
                    prefix::Mixed mix{};
                    CHECK(mix_prefix(b.d, prm, dim3(8, 1, 1), &mix) == GLA_OK, "mix");
                    int64_t want = 0;
                    const int64_t tile = 16 * prefix_tiles(b.d);
                    for (int n : sizes) want += ((int64_t)n * (s.heads / s.kv_heads) + tile - 1) / tile;
                    want *= (int64_t)s.kv_heads * b.d.pre.n_splits;
                    CHECK(host ? mix.n_prefix == want : mix.n_prefix >= want, "%d workgroups for %lld, %d groups", mix.n_prefix,
                          (long long)want, (int)sizes.size());
                    CHECK((int64_t)b.d.pre.split_pages * b.d.pre.n_splits >= b.d.pre.max_prefix / 16 && b.d.pre.split_pages <= 256 &&
                              b.d.pre.max_prefix >= 4096, "splits of %d pages", b.d.pre.split_pages);
                }
    return 0;
}

// A row reads the partials of those splits that hold some of what it sees of the prefix, all of them in the launch, and a
// launch that knows the windows begins with the first that any row sees.
int windows() {
    for (bool host : {false, true})
        for (int own : {1, 30, 500, 4200})
            for (int window : {0, 16, 200, 1024, 4096})
                for (const auto &sizes : {std::vector<int>{16}, {5, 20, 2}}) {
                    std::vector<int32_t> lens{8192, 3000, 900};
                    lens.resize(sizes.size());
                    Batch b(kShapes[1], true, sizes, lens, own, host, window);
                    b.plan();
                    const PrefixLaunch &pre = b.d.pre;
                    if (pre.n_groups == 0) continue;
                    std::set<int> used;
                    for (int r = 0, g = 0; r < b.d.n_seqs; r++) {
                        while (b.starts[g + 1] <= r) g++;
                        const int positions = prefix_positions(b.prefix[g], pre.max_prefix), from = b.start[r];
                        const Splits mine = prefix_splits(pre, positions, from, from + b.len[r]);
                        std::set<int> want, got;
                        for (int j = from; j < positions && j < from + b.len[r]; j++) want.insert(j / 16 / pre.split_pages);
                        for (int i = mine.first; i < mine.first + mine.n; i++) got.insert(i + pre.first_split);
                        CHECK(got == want && (mine.n == 0 || (mine.first >= 0 && mine.first + mine.n <= pre.n_splits)),
                              "row %d of window %d, %d of its own", r, window, own);
                        used.insert(got.begin(), got.end());
                    }
                    if (host)
                        CHECK(used.empty() ? pre.n_splits == 0 : pre.n_splits == *used.rbegin() - *used.begin() + 1,
                              "%d splits, window %d, %d of the rows' own", pre.n_splits, window, own);
                }
    return 0;
}

// Whether the prefixes are read apart: what rows share counts, not what they have.
int rule() {
    const std::vector<int> lone64(64, 1);
    for (bool q8 : {false, true})
        for (bool host : {false, true}) {
            const auto apart = [&](const Shape &s, const std::vector<int> &sizes, const std::vector<int32_t> &lens, int own,
                                   int window = 0, int more = 0) {
                Batch b(s, q8, sizes, lens, own, host, window, more);
                b.plan();
                return b.d.pre.n_groups > 0;
            };
            for (const Shape &s : kShapes) {
                CHECK(apart(s, {64}, {8192}, 500), "64 rows behind 8,192");
                CHECK(apart(s, {10, 4, 10}, {4096, 3000, 2000}, 100), "three groups");
                CHECK(!apart(s, {4}, {128}, 20), "4 rows behind 128");
                CHECK(!apart(s, {64}, {8}, 500), "less than a page");
                CHECK(!apart(s, {2}, {512}, 2000, 0, 62), "a pair among 64 rows of 2,000");
                CHECK(!apart(s, {1, 1, 1}, {4096, 4096, 4096}, 10), "rows alone behind prefixes");
                if (host) CHECK(!apart(s, {8}, {32768}, 4200, 4096), "windows behind the prefix");
            }
            if (!host) {  // bounds of every replay: rows whose own part may grow far beyond what they share
                for (const Shape &s : kShapes) {
                    Batch b(s, q8, {32}, {2048}, 20, false);
                    b.d.pre.max_own = b.d.max_kv_len = 32768;
                    b.plan();
                    CHECK(b.d.pre.n_groups == 1, "a captured call of 32 rows behind 2,048");
                }
            }
            std::vector<int> sizes(64, 1);
            sizes.push_back(2);
            std::vector<int32_t> lens(64, 1024);
            lens.push_back(64);
            CHECK(!apart(kShapes[1], sizes, lens, 50), "lone rows and a pair that shares 64");
            CHECK(apart(kShapes[1], std::vector<int>(32, 2), std::vector<int32_t>(32, 2048), 50), "32 pairs");
        }
    return 0;
}

// The pages of a split that hold a position of [lo, hi), shared out to the waves.
int pages() {
    for (int from : {0, 8, 40})
        for (int n : {0, 1, 2, 7, 8, 33, 256})
            for (int lo : {0, 1, 15, 16, 17, 130, 640, 700, 0x7fffffff})
                for (int hi : {0, 1, 16, 17, 129, 641, 0x7fffffff}) {
                    int a = from, z = from + n;
                    prefix::seen_pages(a, z, lo, hi);
                    std::set<int> want, got[2];
                    for (int p = from; p < from + n; p++)
                        if (lo < hi && p * 16 < hi && p * 16 + 16 > lo) want.insert(p);
                    for (int wave = 0; wave < 4; wave++)
                        for (int even = 0; even < 2; even++) {
                            const prefix::Pages w = even ? prefix::wave_pages<true>(a, z, wave) : prefix::wave_pages<false>(a, z, wave);
                            CHECK(w.n <= 64, "%d pages a wave", w.n);
                            for (int i = 0; i < w.n; i++)
                                CHECK(got[even].insert(w.first + i).second, "page %d twice", w.first + i);
                        }
                    if (lo < hi) CHECK(got[0] == want && got[1] == want, "pages of %d + %d in [%d, %d)", from, n, lo, hi);
                }
    return 0;
}

}  // namespace

int main() {
    if (tiles() || rule() || windows() || pages()) return 1;
    printf("plan ok\n");
    return 0;
}
