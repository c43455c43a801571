// Walks the index arithmetic of the paged kernels (fpga_qwen_b200/csrc/paged.cuh) on the CPU, the way
// the kernels do: every block of every unit is taken by exactly one warp, at most two units of a
// warp's part and of a range are shared, the parts and records of every shared unit are found
// again in order, and every place and every workspace index lies inside its buffer. Prints "ok" or the first violation.
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

// One part of a unit that a warp does not finish alone, and the record of a range.
struct Part { long long off = -1; long long g = 0; int cnt = 0, nblk = 0; };

static void walk(const std::vector<int>& lengths, int cols, int shift, int layers, int hkv, int max_ctas, int min_blocks,
                 int warps) {
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
    long long seen = 0, whole_blocks = 0;
    std::map<std::pair<int, int>, Part> record;                 // (range, slot)
    for (int c = 0; c < sp.ctas; ++c) {
        const long long c0 = sp.begin(c), c1 = sp.begin(c + 1);
        CHECK(c0 < c1 && c0 == seen && c1 - c0 <= 1 << 28);
        CHECK(sp.range_of(c0) == c && sp.range_of(c1 - 1) == c);
        const int blocks = (int)(c1 - c0);
        std::vector<Part> parts(warps * 2);
        for (int w = 0; w < warps; ++w) {
            const long long g0 = c0 + blocks * w / warps, g1 = c0 + blocks * (w + 1) / warps;
            CHECK(g0 == seen);
            if (g0 >= g1) continue;
            PagedUnit u = paged_unit_of(start.data(), n, hkv, g0);
            for (long long g = g0; g < g1;) {
                if (g != g0) paged_next_unit(start.data(), n, hkv, u);
                const PagedUnit x = paged_unit_of(start.data(), n, hkv, g);
                CHECK(x.l == u.l && x.b == u.b && x.kh == u.kh && x.nblk == u.nblk && x.off == u.off);
                CHECK(u.l >= 0 && u.l < layers && u.b >= 0 && u.b < n && u.kh >= 0 && u.kh < hkv && u.nblk > 0);
                CHECK(u.off <= g && g < u.off + u.nblk);
                CHECK(paged_unit_offset(start.data(), n, hkv, u.l, u.b, u.kh) == u.off);
                const long long cnt = std::min(u.off + u.nblk, g1) - g;
                const int t_last = ((int)(g - u.off + cnt) - 1) * PAGED_BLK;
                CHECK(t_last < lengths[u.b] && (t_last >> shift) < cols);
                if (cnt == u.nblk) {
                    whole_blocks += cnt;
                } else {
                    Part& p = parts[w * 2 + (g != g0)];
                    CHECK(p.off < 0);
                    p.off = u.off; p.g = g; p.cnt = (int)cnt; p.nblk = u.nblk;
                }
                seen += cnt;
                g += cnt;
            }
        }
        for (int i = 0; i < warps * 2;) {                       // the merge of the warps' parts
            if (parts[i].off < 0) { ++i; continue; }
            Part sum = parts[i];
            sum.cnt = 0;
            for (; i < warps * 2; ++i) {
                if (parts[i].off < 0) continue;
                if (parts[i].off != sum.off) break;
                CHECK(parts[i].g == sum.g + sum.cnt);
                sum.cnt += parts[i].cnt;
            }
            if (sum.cnt == sum.nblk) whole_blocks += sum.cnt;
            else CHECK(record.emplace(std::make_pair(c, sum.g != c0 ? 1 : 0), sum).second);
        }
    }
    CHECK(seen == sp.total);
    std::map<std::pair<int, int>, Part> left = record;
    for (const auto& r : record) {                              // the join: by the unit's first range, in order
        const Part& p = r.second;
        const int first = sp.range_of(p.off), nrec = sp.range_of(p.off + p.nblk - 1) - first + 1;
        CHECK(nrec >= 2 && first <= r.first.first && r.first.first < first + nrec);
        if (first != r.first.first) continue;
        long long at = p.off;
        for (int i = 0; i < nrec; ++i) {
            const auto it = left.find({first + i, i == 0 && p.off != sp.begin(first) ? 1 : 0});
            CHECK(it != left.end() && it->second.off == p.off && it->second.g == at);
            at += it->second.cnt;
            left.erase(it);
        }
        CHECK(at == p.off + p.nblk);
        whole_blocks += p.nblk;
    }
    CHECK(left.empty() && whole_blocks == sp.total);            // every unit finished once
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
                        walk(valid, cols, shift, layers, hkv, 148, 8, 8);
                        walk(valid, cols, shift, layers, hkv, pick(1, 600), pick(1, 16), pick(1, 16));
                    }
    // calls of few units: every unit once, its logits in a place of their own inside the workspace,
    // its blocks split over its CTAs and their warps
    for (int n : {1, 3, 18, 148})
        for (int layers : {1, 2, 28})
            for (int hkv : {1, 2, 4, 8})
                for (int most : {1, 7, 8, 32, 33, 64, 255, 256, 257, 5000}) {
                    const int units = n * layers * hkv, ctas = paged_ctas_alone(units, most, 148, 8);
                    CHECK(ctas == 0 || ctas == 1 || ctas == 2 || ctas == 4);
                    if (!ctas) continue;
                    CHECK(units * ctas <= 148 && most <= ctas * 32);
                    std::vector<int> hit(units, 0);
                    for (int i = 0; i < units; ++i) {
                        const PagedUnit u = paged_unit_alone(i, n, hkv, most);
                        CHECK(u.l >= 0 && u.l < layers && u.b >= 0 && u.b < n && u.kh >= 0 && u.kh < hkv);
                        CHECK((u.l * n + u.b) * hkv + u.kh == i && u.off == (long long)i * most);
                        CHECK(u.off + most <= (long long)n * layers * hkv * most);
                        ++hit[(u.l * n + u.b) * hkv + u.kh];
                    }
                    for (int h : hit) CHECK(h == 1);
                    for (int nblk : {1, 2, most / 2 + 1, most}) {
                        if (nblk > most) continue;
                        int at = 0;
                        for (int r = 0; r < ctas; ++r) {
                            const int from = nblk * r / ctas, blocks = nblk * (r + 1) / ctas - from;
                            for (int w = 0; w < 8; ++w) {
                                CHECK(from + blocks * w / 8 == at);
                                at = from + blocks * (w + 1) / 8;
                            }
                        }
                        CHECK(at == nblk);
                    }
                }
    // calls of one sequence: CTAs that fit the GPU at once (two per SM where they have half the warps), and the
    // same split of a unit's blocks over them and their warps
    for (int layers = 1; layers <= 64; ++layers)
        for (int hkv : {1, 2, 4, 8})
            for (int most : {1, 2, 7, 8, 31, 32, 33, 64, 129, 249, 256, 513, 8192, 65536}) {
                const int units = layers * hkv;
                const PagedAlone p = paged_alone_equal(units, most, 148, 8);
                CHECK((p.ctas == 0 && p.warps == 8) || (p.warps == 8 && (p.ctas == 1 || p.ctas == 2 || p.ctas == 4) && units * p.ctas <= 148) ||
                      (p.warps == 4 && p.ctas == 1 && units <= 296));
                CHECK(p.ctas != 4 || units * 4 <= 128);
                CHECK(units > 148 || most > 8 || p.ctas == 1);
                CHECK(units <= 296 || p.ctas == 0);
                if (p.ctas == 0) continue;
                for (int nblk : {1, most / 2 + 1, most}) {
                    int at = 0;
                    for (int k = 0; k < p.ctas; ++k) {
                        const int from = nblk * k / p.ctas, blocks = nblk * (k + 1) / p.ctas - from;
                        for (int w = 0; w < p.warps; ++w) {
                            CHECK(from + blocks * w / p.warps == at);
                            at = from + blocks * (w + 1) / p.warps;
                        }
                    }
                    CHECK(at == nblk);
                }
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
