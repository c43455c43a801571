// paged.cuh — index arithmetic of the paged KV cache, shared by its kernels and by the host test
// that walks it (every division of work and every place in a pool is computed here).
#pragma once

#include <cmath>
#include <cstdint>
#include <cstring>

#ifdef __CUDACC__
#define QA_HD __host__ __device__ __forceinline__
#else
#define QA_HD inline
#endif

namespace qattn {

// Codes left in the error block's ERR_DATA word for page tables, lengths and positions read on the device
// (reported as QA_ERR_INVALID).
constexpr int PAGED_BAD_LENGTH = 61, PAGED_BAD_PAGE = 62, PAGED_BAD_POSITION = 63, PAGED_BAD_SEQ = 64;

// A length as the kernels use it: one outside its table (cols pages of 1 << shift rows) is 0.
QA_HD int paged_length(int len, int cols, int shift) { return len < 0 || len > cols << shift ? 0 : len; }

// Page of a new row that its sequence `seq` holds as its len-th, or -1 with *code set (0: a padded row).
QA_HD int paged_place(int len, int seq, int pos, int n_seqs, int cols, int shift, int rope_rows, int n_pages,
                      const int* table, int* code) {
    *code = 0;
    if (len == 0) return -1;
    if ((unsigned)pos >= (unsigned)rope_rows) { *code = PAGED_BAD_POSITION; return -1; }
    if ((unsigned)seq >= (unsigned)n_seqs) { *code = PAGED_BAD_SEQ; return -1; }
    const unsigned col = ((unsigned)len - 1u) >> shift;
    if (col >= (unsigned)cols) { *code = PAGED_BAD_LENGTH; return -1; }
    const int page = table[(size_t)seq * cols + col];
    if ((unsigned)page >= (unsigned)n_pages) { *code = PAGED_BAD_PAGE; return -1; }
    return page;
}

// ---- even split of an attention call --------------------------------------------------------------
// The 16-row blocks of all units (layer, row, KV head), laid end to end in that order, are cut
// into `ctas` equal ranges. start[b] = blocks of one head of rows [0, b), b <= n.
constexpr int PAGED_BLK = 16;                 // cache rows per block (the smallest page)

struct PagedUnit { int l, b, kh, nblk; long long off; };   // blocks [off, off + nblk) of the call

// a / b of non-negative values; a 64-bit division costs the kernels' prologues some hundred cycles.
QA_HD long long paged_div(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

struct PagedSplit {
    long long total, per;                     // blocks of the call; of a range, the first `rem` of which hold one more
    int ctas, rem;                            // ranges in use
    QA_HD long long begin(int c) const { return c * per + (c < rem ? c : rem); }
    QA_HD int range_of(long long g) const {   // range that holds block g
        const long long edge = rem * (per + 1);
        return (int)(g < edge ? paged_div(g, per + 1) : rem + paged_div(g - edge, per));
    }
};

QA_HD PagedSplit paged_split(long long total, int max_ctas, int min_blocks) {
    PagedSplit s;
    s.total = total;
    const long long fit = paged_div(total, min_blocks);
    s.ctas = fit < 1 ? 1 : fit < max_ctas ? (int)fit : max_ctas;
    s.per = paged_div(total, s.ctas);
    s.rem = (int)(total - s.per * s.ctas);
    return s;
}

// First block of unit (l, b, kh).
QA_HD long long paged_unit_offset(const int* start, int n, int hkv, int l, int b, int kh) {
    return (long long)hkv * start[n] * l + (long long)hkv * start[b] + (long long)kh * (start[b + 1] - start[b]);
}

QA_HD PagedUnit paged_unit_of(const int* start, int n, int hkv, long long g) {
    const long long layer_blocks = (long long)hkv * start[n];
    PagedUnit u;
    u.l = (int)paged_div(g, layer_blocks);
    const long long r = g - u.l * layer_blocks;
    int lo = 0, hi = n;                       // largest b with hkv * start[b] <= r (rows of length 0 have no width)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((long long)hkv * start[mid] <= r) lo = mid; else hi = mid;
    }
    u.b = lo;
    u.nblk = start[lo + 1] - start[lo];
    const long long rr = r - (long long)hkv * start[lo];
    u.kh = (int)paged_div(rr, u.nblk);
    u.off = g - (rr - (long long)u.kh * u.nblk);
    return u;
}

// The unit after u; not called past the last one.
QA_HD void paged_next_unit(const int* start, int n, int hkv, PagedUnit& u) {
    u.off += u.nblk;
    if (++u.kh == hkv) {
        u.kh = 0;
        do {
            if (++u.b == n) { u.b = 0; ++u.l; }
            u.nblk = start[u.b + 1] - start[u.b];
        } while (u.nblk == 0);
    }
}

// Calls of few units: unit i (of n_layers * n * hkv) has CTAs of its own, and its blocks begin at
// i * most, where `most` is the blocks that a table row can hold. `nblk` is filled by the caller.
QA_HD PagedUnit paged_unit_alone(int i, int n, int hkv, int most) {
    PagedUnit u;
    const int lb = i / hkv;
    u.kh = i - lb * hkv;
    u.l = lb / n;
    u.b = lb - u.l * n;
    u.nblk = 0;
    u.off = (long long)i * most;
    return u;
}
// CTAs of each unit in such a call (1, 2 or 4; of `warps` warps), or 0: the even split. By estimated
// times in units of 0.095 us, measured over 8 to 144 units of 1 to 8192 rows: a launch of its own
// CTAs 44, a cluster's join 18, a block of every warp 10; the even split with its second launch 92,
// and 13 for each block that its warps have past the first. `most` is the longest row that the
// table can hold, so a warp gets at most four blocks (ragged lengths leave CTAs idle), and clusters
// of four take at most 128 SMs (GPCs do not hold a multiple of four).
QA_HD int paged_ctas_alone(long long units, int most, int max_ctas, int warps) {
    if (units > max_ctas) return 0;
    const long long x = units * most * 10 / ((long long)max_ctas * warps);      // blocks per warp, in tenths
    long long best = 92 + (x > 9 ? (x - 9) * 13 / 10 : 0);
    int ctas = 0;
    for (int k = 1; k <= 4; k *= 2) {
        if (units * k > (k == 4 ? max_ctas - 20 : max_ctas) || most > k * warps * 4) continue;
        const long long cost = 44 + (k > 1 ? 18 : 0) + (long long)most * 10 / (k * warps);
        if (cost < best) { best = cost; ctas = k; }
    }
    return ctas;
}

// The same for a call of one sequence, whose units are equally long: a CTA of its own is never held up by a
// longer neighbour, so there is no limit on rows, and up to two units per SM go side by side in CTAs of
// half the warps. In the same units of time, measured over 8 to 224 units of 512 to 8192 rows: a block of
// every warp 10, or what HBM needs for all warps of the call (14.6 where they fill the GPU); the even
// split 15 for each block that its warps have past the first (160 units of 2048 rows: 33.4 us either
// way, of 1024 rows 19.0 against 21.4).
struct PagedAlone { int ctas, warps; };
QA_HD PagedAlone paged_alone_equal(long long units, int most, int max_ctas, int warps) {
    PagedAlone got{0, warps};
    if (units > 2 * max_ctas) return got;
    const long long all = (long long)max_ctas * warps, x = units * most * 10 / all;
    long long best = 92 + (x > 10 ? (x - 10) * 15 / 10 : 0);
    auto offer = [&](int k, int w) {
        const long long used = units * k * w, hbm = 146 * used / all;      // in tenths
        const long long cost = 44 + (k > 1 ? 18 : 0) + (hbm > 100 ? hbm : 100) * most / (10 * k * w);
        if (cost < best) { best = cost; got = PagedAlone{k, w}; }
    };
    if (units > max_ctas) { offer(1, warps / 2); return got; }
    for (int k = 1; k <= 4; k *= 2)
        if (units * k <= (k == 4 ? max_ctas - 20 : max_ctas)) offer(k, warps);
    return got;
}

// ---- eviction order -------------------------------------------------------------------------------
// Larger weight <=> larger key; -0 equals 0; NaN is the lowest.
QA_HD uint32_t evict_key(float w) {
    if (w != w) return 0u;
    w += 0.f;
    uint32_t b;
#ifdef __CUDA_ARCH__
    b = __float_as_uint(w);
#else
    std::memcpy(&b, &w, 4);
#endif
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

}  // namespace qattn
