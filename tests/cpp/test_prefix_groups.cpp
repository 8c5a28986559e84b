// Groups of sequences that begin with the same pages (group_prefixes), against every way to cut small batches.
#include "../../glint_amd/host/prefix_groups.hpp"

#include <cstdio>
#include <random>

using glint::PrefixGroups;
typedef std::vector<std::vector<int32_t>> Tables;

static PrefixGroups groups(const Tables &t) {
    std::vector<const std::vector<int32_t> *> p;
    for (const auto &x : t) p.push_back(&x);
    return glint::group_prefixes(p);
}

static size_t shared(const Tables &t, size_t a, size_t end) {
    size_t n = 0;
    for (;; n++)
        for (size_t b = a; b < end; b++)
            if (n >= t[b].size() || t[b][n] != t[a][n]) return n;
}

// Pages saved by groups that end where `cuts` has a bit.
static size_t saved(const Tables &t, unsigned cuts) {
    size_t sum = 0;
    for (size_t a = 0, b = 0; b < t.size(); b++)
        if (b + 1 == t.size() || (cuts >> b & 1)) {
            if (b > a) sum += (b - a) * shared(t, a, b + 1);
            a = b + 1;
        }
    return sum;
}

static int check(const Tables &t, const char *what) {
    const PrefixGroups g = groups(t);
    bool ok = g.start.front() == 0 && g.start.back() == (int32_t)t.size() && g.start.size() == g.pages.size() + 1;
    size_t mine = 0, best = 0;
    for (size_t i = 0; ok && i < g.pages.size(); i++) {
        const size_t a = (size_t)g.start[i], end = (size_t)g.start[i + 1];
        ok = a < end && (size_t)g.pages[i] == (end - a > 1 ? shared(t, a, end) : 0);
        mine += (end - a - 1) * (size_t)g.pages[i];
    }
    for (unsigned cuts = 0; !t.empty() && cuts < 1u << (t.size() - 1); cuts++) best = std::max(best, saved(t, cuts));
    if (ok && mine == best) return 0;
    std::printf("%s: %zu pages saved, %zu can be\n", what, mine, best);
    for (size_t i = 0; i < g.pages.size(); i++) std::printf("  rows %d .. share %d\n", g.start[i], g.pages[i]);
    return 1;
}

// A sequence of `n` pages of document `doc` and `own` more, behind the page that all have.
static std::vector<int32_t> seq(int doc, int n, int own) {
    static int32_t fresh = 1 << 20;
    std::vector<int32_t> t{0};
    for (int i = 0; i < n; i++) t.push_back(1000 * doc + i);
    for (int i = 0; i < own; i++) t.push_back(fresh++);
    return t;
}

int main() {
    int bad = 0;
    bad += check({}, "no rows");
    bad += check({seq(1, 5, 2)}, "one row");
    // a row that has the system prompt alone, before, inside and behind eight forks of a document
    for (int at : {0, 4, 8}) {
        Tables t;
        for (int i = 0; i < 8; i++) t.push_back(seq(1, 300, 1 + i));
        t.insert(t.begin() + at, seq(2, 0, 40));
        bad += check(t, "a lone row beside forks");
        const PrefixGroups g = groups(t);
        int most = 0;
        for (int32_t p : g.pages) most = std::max(most, (int)p);
        if (most != 301) bad++, std::printf("forks share %d pages, not 301\n", most);
    }
    {
        Tables t;
        for (int doc = 1; doc < 5; doc++)
            for (int i = 0; i < 2; i++) t.push_back(seq(doc, 20 * doc, 3));
        bad += check(t, "pairs behind one system prompt");
    }
    std::mt19937 rng(1);
    for (int k = 0; k < 3000 && !bad; k++) {  // prefixes of few kinds, so that rows share much or little
        Tables t;
        for (unsigned n = rng() % 10; t.size() < n;) {
            std::vector<int32_t> x;
            for (unsigned i = rng() % 7; i > 0; i--) x.push_back((int32_t)(rng() % (x.size() < 2 ? 1 : 2)));
            t.push_back(x);
        }
        bad += check(t, "random tables");
    }
    if (!bad) std::printf("groups ok\n");
    return bad != 0;
}
