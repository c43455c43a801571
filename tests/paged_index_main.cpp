// Walks the index arithmetic of the paged kernels (fpga_qwen_b200/csrc/paged.cuh) on the CPU, the way
// the kernels do: every block of every unit is taken by exactly one range, at most two units of a
// range are shared, every shared unit's records are found again by the join, and every place and
// every workspace index lies inside its buffer. Prints "ok" or the first violation.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <map>
#include <random>
#include <vector>

#include "../fpga_qwen_b200/csrc/paged.cuh"

using namespace qattn;

#define CHECK(cond)                                                                   \
    do {                                                                              \
        if (!(cond)) { std::printf("line %d: %s\n", __LINE__, #cond); std::exit(1); } \
    } while (0)

static void walk(const std::vector<int>& lengths, int cols, int shift, int layers, int hkv, int max_ctas, int min_blocks) {
    const int n = (int)lengths.size();
    std::vector<int> start(n + 1, 0);
    for (int b = 0; b < n; ++b) {
        const int len = paged_length(lengths[b], cols, shift);
        CHECK(len >= 0 && len <= cols << shift);
        start[b + 1] = start[b] + (len + PAGED_BLK - 1) / PAGED_BLK;
    }
    const PagedSplit sp = paged_split((long long)layers * hkv * start[n], max_ctas, min_blocks);
    CHECK(sp.ctas >= 1 && sp.ctas <= max_ctas);
    const long long bound = (long long)n * layers * hkv * (((cols << shift) + PAGED_BLK - 1) / PAGED_BLK);
    CHECK(sp.total <= bound);                                   // logits [total * 16][2] fit the workspace
    if (!sp.total) return;
    long long seen = 0;
    std::map<std::pair<int, int>, long long> record;            // (range, slot) -> unit offset
    for (int c = 0; c < sp.ctas; ++c) {
        const long long g0 = sp.begin(c), g1 = sp.begin(c + 1);
        CHECK(g0 < g1 && g0 == seen);
        CHECK(sp.range_of(g0) == c && sp.range_of(g1 - 1) == c);
        PagedUnit u = paged_unit_of(start.data(), n, hkv, g0);
        for (long long g = g0; g < g1;) {
            if (g != g0) paged_next_unit(start.data(), n, hkv, u);
            const PagedUnit w = paged_unit_of(start.data(), n, hkv, g);
            CHECK(w.l == u.l && w.b == u.b && w.kh == u.kh && w.nblk == u.nblk && w.off == u.off);
            CHECK(u.l >= 0 && u.l < layers && u.b >= 0 && u.b < n && u.kh >= 0 && u.kh < hkv && u.nblk > 0);
            CHECK(u.off <= g && g < u.off + u.nblk);
            const long long cnt = std::min(u.off + u.nblk, g1) - g;
            const int t_last = ((int)(g - u.off + cnt) - 1) * PAGED_BLK;
            CHECK(t_last < lengths[u.b] && (t_last >> shift) < cols);
            if (cnt != u.nblk) {
                const int slot = g != g0;
                CHECK(record.emplace(std::make_pair(c, slot), u.off).second);
            }
            seen += cnt;
            g += cnt;
        }
    }
    CHECK(seen == sp.total);
    size_t found = 0;
    for (int c = 0; c < sp.ctas; ++c) {                         // the join
        long long done = -1;
        for (int side = 0; side < 2; ++side) {
            const PagedUnit u = paged_unit_of(start.data(), n, hkv, side ? sp.begin(c + 1) - 1 : sp.begin(c));
            if (u.off == done) continue;
            done = u.off;
            const int first = sp.range_of(u.off), last = sp.range_of(u.off + u.nblk - 1);
            CHECK(first <= c && c <= last);
            if (first == last || c != first) continue;
            for (int r = first; r <= last; ++r) {
                const auto it = record.find({r, r == first && u.off != sp.begin(r) ? 1 : 0});
                CHECK(it != record.end() && it->second == u.off);
                ++found;
            }
        }
    }
    CHECK(found == record.size());                              // every shared unit joined once
}

int main() {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    for (int shift = 4; shift <= 9; ++shift)
        for (int n : {1, 2, 3, 64, 1024})
            for (int layers : {1, 28})
                for (int hkv : {1, 2, 4, 8})
                    for (int rep = 0; rep < 6; ++rep) {
                        const int most = rep == 0 ? 1 : rep == 1 ? 17 : n > 64 ? 300 : n > 3 ? 5000 : rep == 2 ? 1 << 20 : 200000;
                        const int cols = (most + (1 << shift) - 1) >> shift;
                        std::vector<int> len(n);
                        for (int& x : len) x = rep == 3 ? most : pick(rep == 4 ? 0 : 1, most);
                        if (rep == 5)
                            for (int& x : len) x = pick(0, 3) ? 0 : pick(-5, 2 * most);    // outside the table: as empty
                        std::vector<int> valid(len);
                        for (int& x : valid) x = paged_length(x, cols, shift);
                        walk(valid, cols, shift, layers, hkv, 296, 4);
                        walk(valid, cols, shift, layers, hkv, pick(1, 600), pick(1, 16));
                    }
    // places: every combination of bad and good length, sequence, position and page id
    for (int shift = 4; shift <= 9; ++shift) {
        const int cols = 3, n_seqs = 4, n_pages = 7;
        std::vector<int> table(n_seqs * cols);
        for (size_t i = 0; i < table.size(); ++i) table[i] = i == 5 ? 7 : i == 6 ? -1 : (int)(i % n_pages);
        const int edge = cols << shift, big = std::numeric_limits<int>::max(), small = std::numeric_limits<int>::min();
        for (int len : {small, -1, 0, 1, 1 << shift, (1 << shift) + 1, edge, edge + 1, big})
            for (int seq : {small, -1, 0, 1, 2, 3, 4, big})
                for (int pos : {small, -1, 0, 99, 100, big}) {
                    int code = -1;
                    const int page = paged_place(len, seq, pos, n_seqs, cols, shift, 100, n_pages, table.data(), &code);
                    CHECK(page >= -1 && page < n_pages && (page >= 0 ? code == 0 : true));
                    const bool pos_ok = pos >= 0 && pos < 100, seq_ok = seq >= 0 && seq < n_seqs, len_ok = len > 0 && len <= edge;
                    if (len == 0) CHECK(page == -1 && code == 0);
                    else if (!pos_ok) CHECK(page == -1 && code == PAGED_BAD_POSITION);
                    else if (!seq_ok) CHECK(page == -1 && code == PAGED_BAD_SEQ);
                    else if (!len_ok) CHECK(page == -1 && code == PAGED_BAD_LENGTH);
                    else {
                        const int id = table[seq * cols + ((len - 1) >> shift)];
                        CHECK(id >= 0 && id < n_pages ? page == id && code == 0 : page == -1 && code == PAGED_BAD_PAGE);
                    }
                }
    }
    // eviction order
    const float inf = std::numeric_limits<float>::infinity(), nan = std::numeric_limits<float>::quiet_NaN();
    const std::vector<float> up = {nan, -inf, -3.f, -1e-40f, 0.f, 1e-45f, 1e-3f, 1.f, 3e38f, inf};
    for (size_t i = 0; i < up.size(); ++i)
        for (size_t j = 0; j < up.size(); ++j) CHECK((evict_key(up[i]) < evict_key(up[j])) == (i < j));
    CHECK(evict_key(-0.f) == evict_key(0.f) && evict_key(-nan) == evict_key(nan));
    std::puts("ok");
    return 0;
}
