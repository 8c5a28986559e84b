// The pages that a window with sinks (visible_of) or behind a prefix (host_seq_pages) touches, against every position in
// turn. Host code only.
#include <stdio.h>

#include <set>
#include <vector>

#include "../../glint_amd/csrc/gla_internal.h"

static int check(int start, int len, int max_len, int limit, int sinks) {
    const gla::Visible v = gla::visible_of(start, len, max_len, limit, sinks);
    const long s = start < 0 ? 0 : start;
    const long n = len < 0 ? 0 : (len > max_len ? max_len : len);
    const long e = s + n < limit ? s + n : limit;
    std::set<int> want;
    for (long j = 0; j < e; j++)
        if (s < e && (j >= s || j < sinks)) want.insert((int)(j / 16));
    std::vector<int> got;
    for (int i = 0; i < v.n_pages; i++) got.push_back(v.page(i));
    if (got != std::vector<int>(want.begin(), want.end())) {
        printf("pages of start %d len %d max %d limit %d sinks %d\n", start, len, max_len, limit, sinks);
        return 1;
    }
    gla::DecodeLaunch d{};
    d.max_kv_len = max_len;
    d.n_sinks = sinks;
    d.pm.pos_limit = limit;
    if (v.n_pages > gla::max_window_pages(d)) {
        printf("%d pages, more than %d\n", v.n_pages, gla::max_window_pages(d));
        return 1;
    }
    for (int p : got) {
        bool all = true;
        for (int j = 16 * p; j < 16 * p + 16; j++) {
            const bool sees = j < e && (j >= s || j < sinks);
            if (v.sees(j) != sees) {
                printf("position %d of start %d len %d sinks %d\n", j, start, len, sinks);
                return 1;
            }
            all = all && sees;
        }
        if (v.whole(p) && !all) {
            printf("page %d of start %d len %d sinks %d\n", p, start, len, sinks);
            return 1;
        }
    }
    return 0;
}

// The pages of a window behind a prefix of `from` positions (host_seq_pages).
static int check_behind(int start, int len, int max_len, int limit, int from) {
    const long s = start < 0 ? 0 : start;
    const long n = len < 0 ? 0 : (len > max_len ? max_len : len);
    const long e = s + n < limit ? s + n : limit;
    std::set<int> want;
    for (long j = from > s ? from : s; j < e; j++) want.insert((int)(j / 16));
    if (gla::host_seq_pages(start, len, max_len, limit, from) == (int)want.size()) return 0;
    printf("pages of start %d len %d max %d limit %d from %d\n", start, len, max_len, limit, from);
    return 1;
}

int main() {
    for (int limit : {1, 16, 100, 160})
        for (int start = -2; start < 110; start += start < 36 ? 1 : 7)
            for (int len = -1; len < 120; len += len < 36 ? 1 : 11)
                for (int max_len : {0, 30, 119}) {
                    for (int sinks : {1, 4, 15, 16, 17, 32, 33, 50, 1000})
                        if (check(start, len, max_len, limit, sinks)) return 1;
                    for (int from : {0, 16, 32, 96})
                        if (check_behind(start, len, max_len, limit, from)) return 1;
                }
    const int big = 2147483647;
    for (int sinks : {1, 20, big})
        for (int start : {big, big - 5, 90})
            if (check(start, big, big, 160, sinks)) return 1;
    printf("pages ok\n");
    return 0;
}
