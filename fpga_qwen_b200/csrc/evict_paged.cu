// evict_paged.cu — eviction from a paged KV cache by accumulated attention weight.
//
// Per unit (sequence, layer, KV head) with L rows and keep < L: the last `recent` rows stay, and of
// the L - recent older ones the keep - recent with the largest weights (ties: the lower row; NaN
// below everything). Selection is a radix search of the threshold over order-preserving 32-bit
// keys, eight bits a pass; then one ascending scan writes the kept rows' indices and moves their
// weights. A second launch moves the K and V rows.
//
// Both moves go forward in tiles: the j-th kept row's old index is at least j, so a tile's
// destinations lie at or below every later tile's sources, and a barrier between a tile's loads
// and its stores makes the move safe in place. Columns are independent, so a unit's rows are
// split over CTAs by column slice (not by row).
#include "qattn_common.cuh"

namespace qattn {
namespace {

constexpr int SEL_THREADS = 512, SEL_WARPS = SEL_THREADS / 32;

__device__ __forceinline__ int row_length(const PagedEvictArgs& a, int b) {
    return paged_length(a.lengths[b], a.src_cols, a.kv.shift);
}

// Exclusive scan over the CTA of one count per thread; *total: their sum. s: [SEL_WARPS + 1].
__device__ __forceinline__ int block_scan(int v, int* s, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    __syncthreads();                               // s is free
    if (lane == 31) s[warp] = incl;
    __syncthreads();
    int base = 0, sum = 0;
    #pragma unroll
    for (int w = 0; w < SEL_WARPS; ++w) {
        if (w < warp) base += s[w];
        sum += s[w];
    }
    *total = sum;
    return base + incl - v;
}

__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const PagedEvictArgs a) {
    __shared__ int hist[256], scan[SEL_WARPS];
    __shared__ unsigned s_prefix;
    __shared__ int s_need;
    const int tid = threadIdx.x;
    const int h = blockIdx.x % a.kv.hkv, layer = (blockIdx.x / a.kv.hkv) % a.kv.layers, b = blockIdx.x / (a.kv.hkv * a.kv.layers);
    const int L = row_length(a, b), mask = (1 << a.kv.shift) - 1;
    if (tid == 0 && a.lengths[b] != L) atomicCAS(a.error, 0, PAGED_BAD_LENGTH);
    int* kept = a.kept + (size_t)blockIdx.x * a.keep;
    const int* src = a.src_table + (size_t)b * a.src_cols;
    const int* dst = a.dst_table + (size_t)b * a.dst_cols;
    auto weight_at = [&](int t) {
        const int page = src[t >> a.kv.shift];
        if (!a.kv.has(page)) { atomicCAS(a.error, 0, PAGED_BAD_PAGE); return 0.f; }
        return *a.kv.weight(page, layer, h, t & mask);
    };
    const int old = L - a.recent;                  // rows that compete (when L > keep)
    unsigned prefix = 0;
    int need = a.keep - a.recent;                  // of them to keep
    const bool all = L <= a.keep;
    if (!all && need > 0) {
        // threshold: the key of rank `need`; need becomes the number of rows equal to it to keep
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += SEL_THREADS) hist[i] = 0;
            __syncthreads();
            for (int t = tid; t < old; t += SEL_THREADS) {
                const unsigned k = evict_key(weight_at(t));
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int d = 255;
                while (hist[d] < need) need -= hist[d--];
                s_prefix = prefix | (unsigned)d << shift;
                s_need = need;
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;
        }
    }
    // ---- ascending pass: indices and weights of the kept rows ----
    int out = 0, ties = 0;                         // kept and tied rows before this tile
    for (int t0 = 0; t0 < L; t0 += SEL_THREADS) {
        const int t = t0 + tid;
        float w = 0.f;
        int above = 0, tie = 0;
        if (t < L) {
            w = weight_at(t);
            if (all || t >= old) above = 1;
            else if (a.keep > a.recent) {
                const unsigned k = evict_key(w);
                above = k > prefix;
                tie = k == prefix;
            }
        }
        int n_tie, n_kept;
        const int tie_rank = ties + block_scan(tie, scan, &n_tie);
        const int flag = above || (tie && tie_rank < need);
        const int j = out + block_scan(flag, scan, &n_kept);   // its barriers order the loads above before the stores below
        if (flag) {
            kept[j] = t;
            const int page = dst[j >> a.kv.shift];
            if (a.kv.has(page)) *a.kv.weight(page, layer, h, j & mask) = w;
            else atomicCAS(a.error, 0, PAGED_BAD_PAGE);
        }
        out += n_kept;
        ties += n_tie;
    }
    for (int j = out + tid; j < a.keep; j += SEL_THREADS) kept[j] = -1;
}

constexpr int MOVE_THREADS = 256, UNROLL = 4;

// CTA (unit, K|V, column slice of SLICE 16-byte chunks): moves the kept rows' slices.
template <int SLICE>
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const PagedEvictArgs a) {
    constexpr int ROWS = MOVE_THREADS / SLICE;     // rows per load
    const int unit = blockIdx.x, kv = blockIdx.y, slice = blockIdx.z;
    const int h = unit % a.kv.hkv, layer = (unit / a.kv.hkv) % a.kv.layers, b = unit / (a.kv.hkv * a.kv.layers);
    const int mask = (1 << a.kv.shift) - 1;
    const int chunk = slice * SLICE + threadIdx.x % SLICE, r = threadIdx.x / SLICE;
    const int* kept = a.kept + (size_t)unit * a.keep;
    const int* src = a.src_table + (size_t)b * a.src_cols;
    const int* dst = a.dst_table + (size_t)b * a.dst_cols;
    if (layer == 0 && h == 0 && kv == 0 && slice == 0 && threadIdx.x == 0) {
        int lo = 0, hi = a.keep;                   // kept rows: the first -1
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (kept[mid] >= 0) lo = mid + 1; else hi = mid;
        }
        a.new_lengths[b] = lo;
    }
    for (int j0 = 0; j0 < a.keep; j0 += ROWS * UNROLL) {
        uint4 v[UNROLL];
        bool ok[UNROLL];
        #pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int j = j0 + i * ROWS + r;
            const int t = j < a.keep ? kept[j] : -1;
            ok[i] = false;
            if (t >= 0) {
                const int page = src[t >> a.kv.shift];
                ok[i] = a.kv.has(page);
                if (ok[i]) v[i] = reinterpret_cast<const uint4*>(a.kv.row(page, layer, kv, h, t & mask))[chunk];
            }
        }
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int j = j0 + i * ROWS + r;
            if (ok[i]) {
                const int page = dst[j >> a.kv.shift];
                if (a.kv.has(page)) reinterpret_cast<uint4*>(a.kv.row(page, layer, kv, h, j & mask))[chunk] = v[i];
            }
        }
    }
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvictArgs& a, cudaStream_t s) {
    const int units = a.n * a.kv.layers * a.kv.hkv;
    evict_select_kernel<<<units, SEL_THREADS, 0, s>>>(a);
    evict_move_kernel<2><<<dim3(units, 2, 8), MOVE_THREADS, 0, s>>>(a);
    return cudaSuccess;
}

}  // namespace qattn
