// Neighbouring sequences of a paged batch that begin with the same pages, as gla_decode_shared takes them.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <limits>
#include <vector>

namespace glint {

struct PrefixGroups {
    std::vector<int32_t> start{0};  // rows of group g: [start[g], start[g + 1])
    std::vector<int32_t> pages;     // that they share; 0 for a row alone
};

// The groups that save the most pages, each read once for its group instead of once a row:
// a row that shares one page with a group (a system prompt) must not take it down to that
// page, nor two groups that share it each other. By dynamic programming over the first rows
// of groups, which ends a group where nothing is shared: n^2 steps for n rows of one prefix
// (512 rows 0.1 ms).
inline PrefixGroups group_prefixes(const std::vector<const std::vector<int32_t> *> &tables) {
    const size_t n = tables.size();
    std::vector<size_t> common(n, 0);  // pages that a row's table begins with as the row's before it
    for (size_t b = 1; b < n; b++) {
        const auto &x = *tables[b - 1], &y = *tables[b];
        const auto end = x.begin() + (ptrdiff_t)std::min(x.size(), y.size());
        common[b] = (size_t)(std::mismatch(x.begin(), end, y.begin()).first - x.begin());
    }
    // of the rows before b: the most pages saved, and the first row of the last group
    std::vector<size_t> best(n + 1, 0), first(n + 1, 0);
    for (size_t a = 0; a < n; a++) {
        size_t shared = std::numeric_limits<size_t>::max();
        for (size_t b = a; b < n; b++) {
            if (b > a) shared = std::min(shared, common[b]);
            if (shared == 0) break;
            const size_t saved = best[a] + (b > a ? (b - a) * shared : 0);
            if (saved > best[b + 1] || (b == a && saved == best[b + 1])) best[b + 1] = saved, first[b + 1] = a;
        }
    }
    PrefixGroups g;
    std::vector<size_t> ends;
    for (size_t end = n; end > 0; end = first[end]) ends.push_back(end);
    for (size_t i = ends.size(); i-- > 0;) {
        const size_t a = (size_t)g.start.back(), end = ends[i];
        size_t shared = end - a > 1 ? std::numeric_limits<size_t>::max() : 0;
        for (size_t b = a + 1; b < end; b++) shared = std::min(shared, common[b]);
        g.start.push_back((int32_t)end);
        g.pages.push_back((int32_t)shared);
    }
    return g;
}

}  // namespace glint
