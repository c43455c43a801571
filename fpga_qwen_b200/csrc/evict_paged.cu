// evict_paged.cu — eviction from a paged KV cache by accumulated attention weight.
//
// Per unit (sequence, layer, KV head) with L rows and keep < L: the last `recent` rows stay, and of
// the L - recent older ones the keep - recent with the largest weights (ties: the lower row; NaN
// below everything).
//
// Selection (one CTA per unit): a radix search of the threshold over order-preserving 32-bit keys,
// eight bits a pass (histogram, then a parallel scan from its top bin), then one ascending pass
// that places every kept row: a row's new index is (rows above the threshold before it) +
// min(tied rows before it, ties to keep), so one scan of both counts serves. Where the table has
// at most SEL_THREADS * PER rows the weights stay in registers from the first load on; longer
// caches read them again for each pass (from L2).
//
// The move is bound by HBM (512 bytes read and 512 written per kept row) and goes forward in
// tiles: the j-th kept row's old index is at least j, so a tile's destinations lie at or below
// every later tile's sources, and a barrier between a tile's loads and its stores makes the move
// safe in place. Channels are independent: a unit's K or V rows are split over CTAs by channel
// slice, not by row, and only as far as it takes to fill the GPU (narrow slices cost DRAM
// efficiency).
#include "qattn_common.cuh"

namespace qattn {
namespace {

constexpr int SEL_THREADS = 512, SEL_WARPS = SEL_THREADS / 32;
constexpr int BINS = 256;

__device__ __forceinline__ int row_length(const PagedEvictArgs& a, int b) {
    return paged_length(a.lengths[b], a.src_cols, a.kv.shift);
}

// The thread's rows are tid, tid + SEL_THREADS, ...: PER of them, held in registers (CACHED), or
// as many as there are, in tiles of PER.
template <int PER, bool CACHED>
__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const PagedEvictArgs a) {
    __shared__ int hist[BINS];
    __shared__ int s_scan[BINS / 32], s_bin, s_need;
    __shared__ int s_cnt[PER * SEL_WARPS], s_off[PER * SEL_WARPS + 1];
    static_assert(PER * SEL_WARPS <= SEL_THREADS && PER * SEL_WARPS % 32 == 0, "one scan over the tile's warps");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x % a.kv.hkv, layer = (blockIdx.x / a.kv.hkv) % a.kv.layers, b = blockIdx.x / (a.kv.hkv * a.kv.layers);
    const int L = row_length(a, b), mask = (1 << a.kv.shift) - 1;
    if (tid == 0 && a.lengths[b] != L) atomicCAS(a.error, 0, PAGED_BAD_LENGTH);
    int* kept = a.kept + (size_t)blockIdx.x * a.keep;
    const int* src = a.src_table + (size_t)b * a.src_cols;
    const int* dst = a.dst_table + (size_t)b * a.dst_cols;
    const bool all = L <= a.keep;
    const int old = L - a.recent;                  // rows that compete (unless all stay)

    float w[PER];
    auto load_tile = [&](int t0) {
        int page[PER];
        #pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int t = t0 + i * SEL_THREADS + tid;
            page[i] = t < L ? src[t >> a.kv.shift] : -1;
        }
        #pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int t = t0 + i * SEL_THREADS + tid;
            w[i] = 0.f;
            if (a.kv.has(page[i])) w[i] = *a.kv.weight(page[i], layer, h, t & mask);
            else if (t < L) atomicCAS(a.error, 0, PAGED_BAD_PAGE);
        }
    };
    if (CACHED) load_tile(0);
    unsigned prefix = 0;
    int need = a.keep - a.recent;                  // competing rows to keep
    if (!all && need > 0) {
        // threshold: the key of rank `need`; need becomes the number of rows equal to it to keep
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < BINS) hist[tid] = 0;
            __syncthreads();
            for (int t0 = 0; t0 < old; t0 += SEL_THREADS * PER) {
                if (!CACHED) load_tile(t0);
                #pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const unsigned k = evict_key(w[i]);
                    if (t0 + i * SEL_THREADS + tid < old && (shift == 24 || ((k ^ prefix) >> (shift + 8)) == 0))
                        atomicAdd(&hist[(k >> shift) & (BINS - 1)], 1);
                }
            }
            __syncthreads();
            // thread i: bin BINS - 1 - i; the bin whose count from the top reaches `need`
            int mine = 0, incl = 0;
            if (tid < BINS) {
                mine = incl = hist[BINS - 1 - tid];
                #pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += x;
                }
                if (lane == 31) s_scan[warp] = incl;
            }
            __syncthreads();
            if (tid < BINS) {
                for (int x = 0; x < warp; ++x) incl += s_scan[x];
                if (incl >= need && incl - mine < need) { s_bin = BINS - 1 - tid; s_need = need - (incl - mine); }
            }
            __syncthreads();
            prefix |= (unsigned)s_bin << shift;
            need = s_need;
        }
    }
    // ---- ascending pass: indices and weights of the kept rows ----
    int above0 = 0, ties0 = 0;                     // rows above the threshold, and tied with it, before this tile
    for (int t0 = 0; t0 < L; t0 += SEL_THREADS * PER) {
        if (!CACHED) load_tile(t0);
        unsigned up[PER], tie[PER];                // ballots of the warp
        #pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int t = t0 + i * SEL_THREADS + tid;
            const unsigned k = evict_key(w[i]);
            const bool competes = t < old && !all, wanted = a.keep > a.recent;
            up[i] = __ballot_sync(0xffffffffu, t < L && (competes ? wanted && k > prefix : true));
            tie[i] = __ballot_sync(0xffffffffu, competes && wanted && k == prefix);
            if (lane == 0) s_cnt[i * SEL_WARPS + warp] = __popc(up[i]) | __popc(tie[i]) << 16;   // at most 8192 each
        }
        __syncthreads();                           // every load of the tile is done too: the stores below may overlap it
        // exclusive scan of the PER * SEL_WARPS packed counts, in row order
        int mine = 0, incl = 0;
        if (tid < PER * SEL_WARPS) {
            mine = incl = s_cnt[tid];
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            if (lane == 31) s_scan[warp] = incl;
        }
        __syncthreads();
        if (tid < PER * SEL_WARPS) {
            for (int x = 0; x < warp; ++x) incl += s_scan[x];
            s_off[tid] = incl - mine;
            if (tid == PER * SEL_WARPS - 1) s_off[PER * SEL_WARPS] = incl;
        }
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int t = t0 + i * SEL_THREADS + tid, off = s_off[i * SEL_WARPS + warp];
            const unsigned before = (1u << lane) - 1u;
            const int ties = ties0 + (off >> 16) + __popc(tie[i] & before);
            const int j = above0 + (off & 0xffff) + __popc(up[i] & before) + min(ties, need);
            if ((up[i] >> lane & 1) || ((tie[i] >> lane & 1) && ties < need)) {
                kept[j] = t;
                const int page = dst[j >> a.kv.shift];
                if (a.kv.has(page)) *a.kv.weight(page, layer, h, j & mask) = w[i];
                else atomicCAS(a.error, 0, PAGED_BAD_PAGE);
            }
        }
        above0 += s_off[PER * SEL_WARPS] & 0xffff;
        ties0 += s_off[PER * SEL_WARPS] >> 16;
    }
    for (int j = above0 + min(ties0, need) + tid; j < a.keep; j += SEL_THREADS) kept[j] = -1;
}

constexpr int MOVE_THREADS = 256, UNROLL = 4;

// CTA (unit, K|V, channel slice of SLICE 16-byte chunks): moves the kept rows' slices.
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
    asm volatile("griddepcontrol.wait;" ::: "memory");       // the selection is complete
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
        int from[UNROLL], to[UNROLL];
        #pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int j = j0 + i * ROWS + r;
            from[i] = j < a.keep ? kept[j] : -1;
        }
        #pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int j = j0 + i * ROWS + r;
            const int page = from[i] < 0 ? -1 : src[from[i] >> a.kv.shift];
            to[i] = from[i] < 0 ? -1 : dst[j >> a.kv.shift];
            if (!a.kv.has(page)) to[i] = -1;       // recorded by the selection
            else v[i] = reinterpret_cast<const uint4*>(a.kv.row(page, layer, kv, h, from[i] & mask))[chunk];
        }
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            const int j = j0 + i * ROWS + r;
            if (a.kv.has(to[i])) reinterpret_cast<uint4*>(a.kv.row(to[i], layer, kv, h, j & mask))[chunk] = v[i];
        }
    }
}

template <int SLICE>
cudaError_t launch_move(const PagedEvictArgs& a, int units, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(units, 2, D * 2 / 16 / SLICE); cfg.blockDim = dim3(MOVE_THREADS); cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, evict_move_kernel<SLICE>, a);
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvictArgs& a, cudaStream_t s) {
    const int units = a.n * a.kv.layers * a.kv.hkv;
    const int max_rows = a.src_cols << a.kv.shift;
    if (max_rows <= SEL_THREADS * 2) evict_select_kernel<2, true><<<units, SEL_THREADS, 0, s>>>(a);
    else if (max_rows <= SEL_THREADS * 8) evict_select_kernel<8, true><<<units, SEL_THREADS, 0, s>>>(a);
    else evict_select_kernel<8, false><<<units, SEL_THREADS, 0, s>>>(a);
    const cudaError_t e = cudaPeekAtLastError();
    if (e != cudaSuccess) return e;
    if (units >= 2 * NUM_SMS_B200) return launch_move<16>(a, units, s);
    if (units >= NUM_SMS_B200 / 2) return launch_move<8>(a, units, s);
    return launch_move<2>(a, units, s);
}

}  // namespace qattn
