// evict_paged.cu — eviction from a paged KV cache by accumulated attention weight.
//
// Per unit (sequence, layer, KV head) with L rows and keep < L: the last `recent` rows stay, and of
// the L - recent older ones the keep - recent with the largest weights (ties: the lower row; NaN
// below everything).
//
// Selection: a radix search of the threshold over order-preserving 32-bit keys, eight bits a pass,
// then one ascending pass that places every kept row: a row's new index is (rows above the
// threshold before it) + min(tied rows before it, ties to keep), so one scan of both counts serves.
// It is a chain of latencies and of code that runs once, so barriers are few (a histogram per pass,
// all cleared at the start; every warp scans the bins, and later the counts, for itself) and the
// code is small: weights lie in shared memory, not in registers, and loops stay rolled. (Unrolled
// over registers it took 10 us for 8 units of 1025 rows, most of it fetching instructions.
// Counting two bits at a time without atomics took twice as long as the histograms.) One CTA takes
// a unit; where the table can hold more than 4096 rows, a cluster of CTAs takes it, each a
// contiguous slice of its rows, and histograms and counts are summed over distributed shared
// memory.
//
// The move is bound by HBM (512 bytes read and 512 written per kept row; whole rows at a time, since
// narrow column slices cost DRAM efficiency: 107 us in 64-byte and 154 us in 32-byte slices against
// 88 us in whole rows, for 2048 rows x 224 units). It goes forward in tiles: the j-th kept row's
// old index is at least j, so a tile's destinations lie at or below every later tile's sources,
// and a barrier between a tile's loads and its stores makes the move safe in place. A unit's K
// or V rows are moved by one CTA, or by a cluster where there are few units, whose CTAs each take
// a part of every tile and meet at the cluster's barrier.
#include <cooperative_groups.h>

#include "qattn_common.cuh"

namespace qattn {
namespace {

namespace cg = cooperative_groups;

constexpr int BINS = 256, BATCH = 4;
constexpr int SLICE_ROWS = 4096;                   // of a cluster's CTA, where there are SMs for it
constexpr int MAX_SLICE = 49152;                   // 192 KB of shared memory
constexpr int TABLE_INTS = 1024;                   // page ids of the destination kept in shared memory

__device__ __forceinline__ int row_length(const PagedEvictArgs& a, int b) {
    return paged_length(a.lengths[b], a.src_cols, a.kv.shift);
}

// The cluster's CTAs each take a contiguous slice of the unit's rows, at most as many as s_w holds.
template <int SEL_THREADS>
__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const PagedEvictArgs a) {
    constexpr int SEL_WARPS = SEL_THREADS / 32;
    extern __shared__ __align__(16) float s_w[];             // the slice's weights
    __shared__ __align__(16) int hist[4][BINS];
    __shared__ __align__(16) int bins[2][BINS];              // of the whole cluster, by turns
    __shared__ int s_dst[TABLE_INTS];
    __shared__ int s_cnt[SEL_WARPS], s_total;                // packed counts: above the threshold, tied << 16
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
    const int unit = blockIdx.x / ranks;
    const int h = unit % a.kv.hkv, layer = (unit / a.kv.hkv) % a.kv.layers, b = unit / (a.kv.hkv * a.kv.layers);
    // What ran before is complete. (No read-only loads below: they may move across this. Launched ahead like
    // the move: one layer of 1025 rows 11.1 -> 10.2 us.)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int L = row_length(a, b), mask = (1 << a.kv.shift) - 1;
    int* kept = a.kept + (size_t)unit * a.keep;
    const int* src = a.src_table + (size_t)b * a.src_cols;
    const int* dst = a.dst_table + (size_t)b * a.dst_cols;
    const bool all = L <= a.keep;
    const int old = all ? 0 : L - a.recent;                  // rows that compete
    const int per = (L + ranks - 1) / ranks;
    const int row0 = min(rank * per, L), rows = min(L - row0, per), compete = min(max(old - row0, 0), rows);

    for (int i = tid; i < 4 * BINS; i += SEL_THREADS) hist[0][i] = 0;
    const int dst_used = ((a.keep - 1) >> a.kv.shift) + 1;
    if (dst_used <= TABLE_INTS) {
        for (int i = tid; i < dst_used; i += SEL_THREADS) s_dst[i] = dst[i];
        dst = s_dst;
    }
    if (tid == 0 && rank == 0 && a.lengths[b] != L) atomicCAS(a.error + ERR_DATA, 0, PAGED_BAD_LENGTH);
    #pragma unroll 1
    for (int i0 = tid; i0 < rows; i0 += SEL_THREADS * BATCH) {
        // all page ids of a batch, then all its weights, in flight at once
        int page[BATCH];
        float w[BATCH];
        #pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int i = i0 + k * SEL_THREADS;
            page[k] = i < rows ? src[(row0 + i) >> a.kv.shift] : 0;
        }
        int bad = 0;
        #pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int i = i0 + k * SEL_THREADS;
            const bool ok = a.kv.has(page[k]);
            bad |= !ok;
            w[k] = ok && i < rows ? *a.kv.weight(page[k], layer, h, (row0 + i) & mask) : 0.f;
        }
        if (bad) atomicCAS(a.error + ERR_DATA, 0, PAGED_BAD_PAGE);
        #pragma unroll
        for (int k = 0; k < BATCH; ++k)
            if (i0 + k * SEL_THREADS < rows) s_w[i0 + k * SEL_THREADS] = w[k];
    }
    __syncthreads();
    // prefix: the threshold, the key of rank `need`; need: first the competing rows to keep, then those
    // of them equal to the threshold
    unsigned prefix = 0;
    int need = all ? 0 : a.keep - a.recent;
    const bool wanted = need > 0;
    #pragma unroll 1
    for (int pass = 0; pass < 4 && wanted; ++pass) {
        const int shift = 24 - 8 * pass;
        const unsigned known = pass ? ~0u << (shift + 8) : 0u;
        #pragma unroll 2
        for (int i = tid; i < compete; i += SEL_THREADS) {
            const unsigned k = evict_key(s_w[i]);
            if (((k ^ prefix) & known) == 0) atomicAdd(&hist[pass][(k >> shift) & (BINS - 1)], 1);
        }
        const int* total = hist[pass];
        if (ranks > 1) {
            cluster.sync();
            if (tid < BINS) {
                int sum = 0;
                #pragma unroll 2
                for (int r = 0; r < ranks; ++r) sum += cluster.map_shared_rank(hist[pass], r)[tid];
                bins[pass & 1][tid] = sum;
            }
            total = bins[pass & 1];
        }
        __syncthreads();
        // lane: bins 255 - 8 lane down to 248 - 8 lane; the bin whose count from the top reaches `need`
        const int4 hi = *reinterpret_cast<const int4*>(total + BINS - 4 - 8 * lane);
        const int4 lo = *reinterpret_cast<const int4*>(total + BINS - 8 - 8 * lane);
        const int v[8] = {hi.w, hi.z, hi.y, hi.x, lo.w, lo.z, lo.y, lo.x};
        int sum = 0;
        #pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i];
        int incl = sum;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        const int at = __ffs(__ballot_sync(0xffffffffu, incl >= need)) - 1;
        int before = incl - sum, bin = BINS - 1 - 8 * lane, in_bin = v[0];
        bool found = false;
        #pragma unroll
        for (int i = 0; i < 7; ++i) {
            found = found || before + v[i] >= need;
            if (!found) { before += v[i]; --bin; in_bin = v[i + 1]; }
        }
        prefix |= (unsigned)__shfl_sync(0xffffffffu, bin, at) << shift;
        need -= __shfl_sync(0xffffffffu, before, at);
        if (need == __shfl_sync(0xffffffffu, in_bin, at) && prefix) {
            --prefix;                                        // the whole bin stays: no need to look inside
            need = 0;
            break;
        }
    }
    // ---- ascending pass: each warp takes a run of the slice's rows; first it counts ----
    const int run = ((rows + SEL_WARPS - 1) / SEL_WARPS + 31) & ~31;
    const int i0 = min(warp * run, rows), i1 = min(i0 + run, rows);
    auto ballots = [&](int i, unsigned& up, unsigned& tie) {
        const unsigned k = i < compete ? evict_key(s_w[i]) : 0u;
        up = __ballot_sync(0xffffffffu, i < i1 && (i < compete ? wanted && k > prefix : true));
        tie = __ballot_sync(0xffffffffu, i < i1 && i < compete && wanted && k == prefix);
    };
    int above = 0, ties = 0;
    #pragma unroll 2
    for (int i = i0 + lane; i - lane < i1; i += 32) {
        unsigned up, tie;
        ballots(i, up, tie);
        above += __popc(up);
        ties += __popc(tie);
    }
    // (a slice holds fewer than 2^16 rows, so both counts fit one word)
    if (lane == 0) s_cnt[warp] = above | ties << 16;
    __syncthreads();
    const int c = lane < SEL_WARPS ? s_cnt[lane] : 0, earlier = lane < warp ? c : 0;
    above = __reduce_add_sync(0xffffffffu, earlier & 0xffff);
    ties = __reduce_add_sync(0xffffffffu, (unsigned)earlier >> 16);
    int all_above = __reduce_add_sync(0xffffffffu, c & 0xffff), all_ties = __reduce_add_sync(0xffffffffu, (unsigned)c >> 16);
    if (ranks > 1) {
        // the slices before this one; this barrier also follows every CTA's loads of weights
        if (tid == 0) s_total = all_above | all_ties << 16;
        cluster.sync();
        const int t = lane < rank ? *cluster.map_shared_rank(&s_total, lane) : 0;
        const int above0 = __reduce_add_sync(0xffffffffu, t & 0xffff), ties0 = __reduce_add_sync(0xffffffffu, (unsigned)t >> 16);
        above += above0; ties += ties0;
        all_above += above0; all_ties += ties0;
    }
    // ---- then it places them ----
    #pragma unroll 2
    for (int i = i0 + lane; i - lane < i1; i += 32) {
        unsigned up, tie;
        ballots(i, up, tie);
        const unsigned before = (1u << lane) - 1u;
        const int my_ties = ties + __popc(tie & before);
        const int j = above + __popc(up & before) + min(my_ties, need);
        if ((up >> lane & 1) || ((tie >> lane & 1) && my_ties < need)) {
            kept[j] = row0 + i;
            const int page = dst[j >> a.kv.shift];
            if (a.kv.has(page)) *a.kv.weight(page, layer, h, j & mask) = s_w[i];
            else atomicCAS(a.error + ERR_DATA, 0, PAGED_BAD_PAGE);
        }
        above += __popc(up);
        ties += __popc(tie);
    }
    if (rank == ranks - 1)                                   // (the last slice's counts are the unit's)
        for (int j = all_above + min(all_ties, need) + tid; j < a.keep; j += SEL_THREADS) kept[j] = -1;
    if (ranks > 1) cluster.sync();                           // until the others have read this CTA's memory
}

constexpr int ROW_THREADS = 8, CHUNKS = 16 / ROW_THREADS;    // threads of a row; 16-byte chunks of a thread
constexpr int PER_THREAD = 2;                                // rows of a thread and tile
constexpr int tile_rows(int threads) { return threads / ROW_THREADS * PER_THREAD; }

// Cluster (unit, K|V): moves the kept rows, tile after tile of TILE rows per CTA. Three tiles are
// under way: one being stored, the next one's rows and the one after's indices and pages being
// loaded. A tile's rows may be loaded before the tile before it is stored, since its sources lie
// above those destinations. Rows that are in place already are not touched. Eight threads take a
// row, two 16-byte chunks each: with sixteen, one chunk each, half of the issue slots went to indices
// and addresses, which cost a few per cent.
template <int MOVE_THREADS>
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const PagedEvictArgs a) {
    constexpr int MOVE_ROWS = MOVE_THREADS / ROW_THREADS, TILE = tile_rows(MOVE_THREADS);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const int unit = blockIdx.x / ranks, kv = blockIdx.y, tile = TILE * ranks;
    const int h = unit % a.kv.hkv, layer = (unit / a.kv.hkv) % a.kv.layers, b = unit / (a.kv.hkv * a.kv.layers);
    const int mask = (1 << a.kv.shift) - 1;
    const int chunk = threadIdx.x % ROW_THREADS, r = rank * TILE + threadIdx.x / ROW_THREADS;
    const int* kept = a.kept + (size_t)unit * a.keep;
    const int* src = a.src_table + (size_t)b * a.src_cols;
    const int* dst = a.dst_table + (size_t)b * a.dst_cols;
    // The selection is complete. (No read-only loads of what it writes: they may move across this.)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (layer == 0 && h == 0 && kv == 0 && rank == 0 && threadIdx.x == 0) {
        int lo = 0, hi = a.keep;                   // kept rows: the first -1
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (kept[mid] >= 0) lo = mid + 1; else hi = mid;
        }
        a.new_lengths[b] = lo;
    }
    int from[PER_THREAD], page[PER_THREAD], to[PER_THREAD];  // of the tile ahead: old row, its page, the new row's page (-1: no move)
    auto load_index = [&](int j0) {
        #pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) {
            const int j = j0 + i * MOVE_ROWS + r;
            from[i] = j < a.keep ? kept[j] : -1;
        }
    };
    auto load_pages = [&](int j0) {
        #pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) {
            const int j = j0 + i * MOVE_ROWS + r;
            page[i] = from[i] < 0 ? -1 : src[from[i] >> a.kv.shift];
            to[i] = from[i] < 0 ? -1 : dst[j >> a.kv.shift];
            if (page[i] == to[i] && ((from[i] ^ j) & mask) == 0) to[i] = -1;   // in place already
        }
    };
    uint4 v[PER_THREAD][CHUNKS], next[PER_THREAD][CHUNKS];
    int dest[PER_THREAD], next_dest[PER_THREAD];   // page to store to, or -1
    auto load_rows = [&](uint4 (&x)[PER_THREAD][CHUNKS], int (&d)[PER_THREAD]) {
        #pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) {
            d[i] = a.kv.has(page[i]) && a.kv.has(to[i]) ? to[i] : -1;      // (bad pages are recorded by the selection)
            if (d[i] >= 0) {
                const uint4* p = reinterpret_cast<const uint4*>(a.kv.row(page[i], layer, kv, h, from[i] & mask)) + chunk;
                #pragma unroll
                for (int k = 0; k < CHUNKS; ++k) x[i][k] = p[k * ROW_THREADS];
            }
        }
    };
    load_index(0);
    load_pages(0);
    load_rows(v, dest);
    load_index(tile);
    load_pages(tile);
    for (int j0 = 0; j0 < a.keep; j0 += tile) {
        load_rows(next, next_dest);                // the tile after this one
        load_index(min(j0 + 2 * tile, a.keep));
        if (ranks > 1) cluster.sync(); else __syncthreads();   // every thread has its rows of this tile
        #pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) {
            const int j = j0 + i * MOVE_ROWS + r;
            if (dest[i] >= 0) {
                uint4* p = reinterpret_cast<uint4*>(a.kv.row(dest[i], layer, kv, h, j & mask)) + chunk;
                #pragma unroll
                for (int k = 0; k < CHUNKS; ++k) p[k * ROW_THREADS] = v[i][k];
            }
            #pragma unroll
            for (int k = 0; k < CHUNKS; ++k) v[i][k] = next[i][k];
            dest[i] = next_dest[i];
        }
        load_pages(j0 + 2 * tile);
    }
}

cudaError_t launch(void (*kernel)(PagedEvictArgs), dim3 grid, int threads, size_t smem, int cluster, bool overlap,
                   const PagedEvictArgs& a, cudaStream_t s) {
    cudaError_t e = cudaSuccess;
    // (the kernel's own most, whatever this call takes: the attribute is the kernel's, and another host thread may be
    // between its own two calls)
    if (smem > 32 << 10) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SLICE * (int)sizeof(float));
    if (e != cudaSuccess) return e;
    if (cluster > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid.x * cluster, grid.y); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cfg.attrs = attr; cfg.numAttrs = overlap ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvictArgs& a, cudaStream_t s) {
    const int units = a.n * a.kv.layers * a.kv.hkv;
    const int max_rows = a.src_cols << a.kv.shift;
    // selection: clusters that bring a slice down to SLICE_ROWS while all of them fit the GPU at once,
    // and in any case to what shared memory holds
    int ranks = 1;
    while (ranks < 16 && max_rows > ranks * SLICE_ROWS &&
           (units * ranks * 2 <= 2 * NUM_SMS_B200 || max_rows > ranks * MAX_SLICE))
        ranks *= 2;
    const int per = (max_rows + ranks - 1) / ranks;
    if (per > MAX_SLICE) return cudaErrorInvalidValue;       // (refused before)
    // short tables: small CTAs, more of them per SM (6,496 units of 65 rows, both
    // launches: 123 -> 61 us; kept 33 of 65: 80 us with a table of 80 rows, 134 us with one of 4096 and 225 us with
    // one of 32768, whose CTAs take the shared memory of a full row: lengths are not known on the host)
    const bool small = per <= 1024 && ranks == 1;
    const cudaError_t e = launch(small ? evict_select_kernel<128> : evict_select_kernel<512>, dim3(units), small ? 128 : 512,
                                 (size_t)per * sizeof(float), ranks, a.overlap, a, s);
    if (e != cudaSuccess) return e;
    // move: clusters that fill the GPU (4 CTAs per SM) where the units alone do not and there are rows
    // for every CTA; where there are many units with few kept rows, small CTAs (224 units of 78 kept rows:
    // 26 -> 18 us)
    ranks = 1;
    while (ranks < 16 && units * 2 * ranks * 2 <= 4 * NUM_SMS_B200 && ranks * tile_rows(256) < a.keep) ranks *= 2;
    if (ranks == 1 && a.keep <= 4 * tile_rows(64)) return launch(evict_move_kernel<64>, dim3(units, 2), 64, 0, 1, true, a, s);
    if (ranks == 1 && a.keep <= 8 * tile_rows(128)) return launch(evict_move_kernel<128>, dim3(units, 2), 128, 0, 1, true, a, s);
    return launch(evict_move_kernel<256>, dim3(units, 2), 256, 0, ranks, true, a, s);
}

}  // namespace qattn
