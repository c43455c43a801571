// attn_paged.cu — decode attention of one query row per sequence over a paged KV cache.
//
// For row b with L = lengths[b] cached rows, layer l and KV head kh, both query heads h of the
// group: s_t = q_h . k_t / sqrt(128), p = softmax(s), out_h = sum_t p_t v_t, all in FP32 over the
// FP16 rows; with add_weights also weights[t] += p_t of both heads.
//
// Bound by HBM: 512 bytes of K and V a row and KV head for 1,024 flops. What keeps HBM busy:
//   * Even split (stream-K style). The 16-row blocks of all (layer, row, KV head) units are laid
//     end to end and cut into equal ranges, one per CTA (one CTA per SM), and a CTA's range again
//     into one part per warp, whatever the lengths are; lengths are read on the device, so every
//     CTA first scans them. A part can end inside one unit and continue in the next.
//   * Every warp is its own pipeline from its first block to its last: one lane keeps STAGES blocks
//     (K and V rows, 8 KB) in flight into the warp's ring with TMA copies (128-byte swizzle),
//     across unit boundaries, 128 KB per SM. A block never crosses a page, so a block is one page
//     id; the next id is loaded one block ahead. No barrier between the warps until all are
//     done: a unit inside a warp's part is finished by the warp alone.
//   * Few instructions per block. With FP32 FMAs a block of 16 rows took about 560 warp
//     instructions (conversions, products, the sum over lanes), about what HBM leaves time for;
//     mma.sync takes K and V as they are and needs a quarter. Both GQA heads share the tile:
//     its N = 8 columns are the FP16 halves (high, low) of both heads' queries, or of both heads'
//     softmax weights, twice. (A tcgen05 tile would hold 128 rows against 16 here and bring TMEM
//     round trips, for no more bytes.)
//
// Numerics: FP16 rows are exact operands. A query (scaled by a power of two so that its largest
// channel lies in [2^13, 2^14)) and a weight (exp2 of the distance to its block's maximum, plus 14) are
// each the sum of two FP16 halves: off by 2^-22 of the value, or by 2^-36 of the largest channel and
// 2^-37 of the block's largest weight, whichever is coarser. Sums are FP32, and long sums are made by
// FMA, with the block's factor (exp2 of the distance of its maximum to the running one): the tensor core's own
// accumulation truncates, which over the hundred blocks of a long history costs a few 2^-20 (2.0e-6 off in
// 2-norm against 64 bits at 131071 rows), so it takes no more than two steps of a chain. The high half is
// rounded towards zero and neither half of a nonzero value is zero, so both have its sign and an infinite key or
// value gives what the formula gives. That adds 2^-37 of the largest to a weight far below it, all of one sign, which is
// why weights are relative to their own block: against the running maximum one heavy row did so to every row after
// it (131071 rows 25 to 80 nats below one, their values 10^5 times as large: outputs off by up to 0.7%, now by
// 1.5e-5, the part of the heavy row's own block; times of whole calls are the same within 1%).
//
// A unit that several warps of a CTA share is merged through shared memory at the CTA's end; a
// unit that several CTAs share leaves one record (max, sum, 2 x 128 partial output) per CTA, and a
// second launch, whose CTAs start behind the first's (programmatic dependent launch), joins
// them in range order: no atomics and no flags, so the result does not depend on timing and the
// workspace needs no initial state. At most two units of a range are shared with other ranges (its
// first and its last), so the records are 2 per CTA, whatever the batch. (Joining in the first
// launch, by the CTA that sees all records of a unit stored, measured slower: its fences and the
// late joins cost 8 us of 81 at 28 layers x 3970 rows.)
//
// The weights need the final maximum and sum: the logits go to the workspace (8 bytes a row and
// KV head against 512 of K and V) and become weights when the unit is finished, by the warp, the
// CTA or, for units shared between CTAs, in the joining launch, each CTA those of its own range.
// Each (row, KV head) weight gets one FP32 addition.
//
// Calls of few units that are not long need none of that: every unit has a CTA, or a cluster of two or
// four, of its own, without the scan of the lengths, and a cluster's CTAs join their parts over
// distributed shared memory, without the second launch (paged_ctas_alone says when: 8 units of 256
// rows 8.6 -> 5.9 us, of 1024 rows 9.0 -> 8.0 us, 32 units of 2048 rows 13.7 -> 10.6 us, 144 units
// of 512 rows 13.7 -> 8.4 us). Neither do calls of one sequence, long or not, whose units are equally
// long: up to 148 of them have CTAs of their own, up to 296 half-size CTAs, two per SM
// (paged_alone_equal: 224 units of 3970 rows 75.1 -> 68.5 us; with weights, of 2049 rows 50.3 -> 42.0 us;
// 112 units of 8192 rows 78.1 -> 71.7 us, all on the same inputs call after call. On inputs that change with every
// call the first is 73 to 74 us, 6.2 TB/s, and the second 47.4 us with the reset of the weights, some 3 us).
// Both rules go by the rows that the table can hold, since lengths are not known on the host; the figures are of
// tables as narrow as the rows. 8 units of 452 rows take 7.3 us with a table of up to 1024 rows and 8.9 us, the
// even split, with a wider one; 64 units of 256 rows 6.5 and 9.3 us.
//
// Every wait is bounded: on expiry the CTA records an error code, consumes no further block, and
// drains its copies before it exits.
#include <cooperative_groups.h>

#include "qattn_common.cuh"
#include "sm100.cuh"

namespace qattn {
namespace {

using namespace sm100;
namespace cg = cooperative_groups;

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int BLK = PAGED_BLK;
constexpr int STAGES = 2;                     // blocks in flight per warp
constexpr int HALF_STAGE = BLK * D * 2;       // K rows, then V rows of a block: 4 KB each, [channel half][row][64]
constexpr int STAGE = 2 * HALF_STAGE;
constexpr int ring_bytes(int warps) { return warps * STAGES * STAGE; }
constexpr int CTAS = NUM_SMS_B200;            // ranges
constexpr int MIN_BLOCKS = WARPS;             // blocks per range, at least
constexpr int JOIN_THREADS = 256, JOIN_GROUPS = JOIN_THREADS / (GROUP * D / 4);
constexpr int JOIN_PARTS = 3;
constexpr int WAIT_CODE = 43;                 // error code of an expired wait

// A part of a unit that its worker does not finish alone.
struct Part {
    int unit;                                 // (l * n + b) * hkv + kh, or -1: none
    int blk0, cnt, nblk;                      // blocks [blk0, blk0 + cnt) of the unit's nblk
    long long g;                              // its first block in the call
    float m[GROUP], l[GROUP];
};
// A unit that a CTA merged: all of its blocks (cnt), or not (0).
struct Whole {
    int unit, cnt;
    long long g;
    float m[GROUP], l[GROUP];
};
// The joining launch's view of a range's part of a shared unit.
struct __align__(16) Shared {
    int nrec, first, first_slot, unit;        // records of the unit (0: no such part), their first range and its slot
    int blk0, cnt;
    long long g;                              // its first block in the call
};
// A CTA's part of its cluster's unit.
struct Joint {
    float o[GROUP * D];
    float m[GROUP], l[GROUP];
    int cnt;                                  // blocks, 0: none
};
__device__ __forceinline__ Shared* shared_of(const PagedAttnArgs& a) { return static_cast<Shared*>(a.shared); }

__device__ __forceinline__ int row_length(const PagedAttnArgs& a, int b) {
    return paged_length(a.lengths[b], a.cols, a.kv.shift);
}

// start[b] = blocks of rows [0, b); called by all threads of the CTA, n <= MAX_PAGED_BATCH.
__device__ __forceinline__ PagedSplit scan_lengths(const PagedAttnArgs& a, int* start, int* warp_sum) {
    constexpr int PER = MAX_PAGED_BATCH / THREADS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int v[PER], sum = 0;
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = tid * PER + i;
        v[i] = sum;
        if (b < a.n) sum += (row_length(a, b) + BLK - 1) / BLK;
    }
    int incl = sum;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int base = incl - sum;
    #pragma unroll
    for (int w = 0; w < WARPS; ++w) base += w < warp ? warp_sum[w] : 0;
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = tid * PER + i;
        if (b < a.n) start[b] = base + v[i];
    }
    if (tid == THREADS - 1) start[a.n] = base + sum;
    __syncthreads();
    return paged_split((long long)a.n_layers * a.kv.hkv * start[a.n], CTAS, MIN_BLOCKS);
}

// exp2(x - m) where m is a maximum that may still be -inf (nothing seen, or only -inf logits).
__device__ __forceinline__ float exp2_from(float x, float m) { return exp2f(x - (m == -INFINITY ? 0.f : m)); }

// weights += p for the rows of blocks [blk0, blk0 + cnt) of a unit of len rows, whose logits begin
// at block g, by threads t of nt, four rows a thread: a vector reduction, which leaves L2 to do the
// addition.
__device__ __forceinline__ void add_weights(const PagedAttnArgs& a, int l, int b, int kh, int len, int blk0, int cnt, long long g,
                                            const float (&M)[GROUP], const float (&L)[GROUP], int t, int nt) {
    const int t0 = blk0 * BLK, rows = min(cnt * BLK, len - t0);
    const float4* s = reinterpret_cast<const float4*>(a.logits + g * (BLK * 2));
    const int* table = a.table + (size_t)b * a.cols;
    const float r0 = 1.f / L[0], r1 = 1.f / L[1];
    #pragma unroll 4
    for (int i = t * 4; i < rows; i += nt * 4) {
        const float4 x = s[i >> 1], y = s[(i >> 1) + 1];
        const int page = table[(t0 + i) >> a.kv.shift];
        const float w[4] = {exp2_from(x.x, M[0]) * r0 + exp2_from(x.y, M[1]) * r1, exp2_from(x.z, M[0]) * r0 + exp2_from(x.w, M[1]) * r1,
                            exp2_from(y.x, M[0]) * r0 + exp2_from(y.y, M[1]) * r1, exp2_from(y.z, M[0]) * r0 + exp2_from(y.w, M[1]) * r1};
        if (!a.kv.has(page)) continue;
        float* dst = a.kv.weight(page, a.layer0 + l, kh, (t0 + i) & ((1 << a.kv.shift) - 1));
        if (i + 4 <= rows)
            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};"
                         ::"l"(dst), "f"(w[0]), "f"(w[1]), "f"(w[2]), "f"(w[3]) : "memory");
        else
            for (int k = 0; k < rows - i; ++k) atomicAdd(dst + k, w[k]);
    }
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// d[16 x 8] += a[16 x 16] b[16 x 8], FP16 operands, FP32 sums.
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b.
__device__ __forceinline__ void mma16816_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// x, |x| < 65504, as high + low FP16 halves (high in the low 16 bits). High is x towards zero; the
// halves of a nonzero x are nonzero and have its sign (the smallest subnormal, 2^-24, where they
// would be zero); infinities and NaN stay in the high half.
__device__ __forceinline__ uint32_t split_half(float x) {
    const uint32_t tiny = x != 0.f ? (__float_as_uint(x) >> 16 & 0x8000u) | 1u : 0u;
    uint32_t hi = __half_as_ushort(__float2half_rz(x));
    const float rest = x - __half2float(__ushort_as_half((unsigned short)hi));
    uint32_t lo = __half_as_ushort(__float2half_rn(rest));
    if (!(fabsf(x) < INFINITY)) return hi;
    if ((hi & 0x7fffu) == 0) hi = tiny;
    if ((lo & 0x7fffu) == 0) lo = tiny;
    return hi | lo << 16;
}

// W warps: WARPS, or fewer for calls whose units each have one CTA (a.alone == 1).
template <bool WEIGHTS, int W = WARPS>
__global__ void __launch_bounds__(W * 32, 1) attn_paged_split_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap map) {
    extern __shared__ __align__(1024) uint8_t ring[];        // [W][STAGES][K rows | V rows]
    constexpr int T = W * 32;
    __shared__ __align__(8) uint64_t full[W][STAGES];
    __shared__ int start[MAX_PAGED_BATCH + 1];
    __shared__ int warp_sum[WARPS];
    __shared__ Part parts[W][2];                             // [0]: of the warp's first unit, [1]: of its last
    __shared__ __align__(16) float s_part[W][2][GROUP * D];
    __shared__ Whole wholes[WEIGHTS ? W * 2 : 1];            // of the merged units, by turn
    __shared__ __align__(16) Joint joint;
    __shared__ int abort_flag, never_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x;
    const int g8 = lane >> 2, j4 = lane & 3, head = j4 & 1;  // tile row or column, and the column pair's head
    const int hkv = a.kv.hkv, alone = W < WARPS ? 1 : a.alone;
    if (tid == 0) {
        abort_flag = 0; never_abort = 0; joint.cnt = 0;
        for (int i = 0; i < W * STAGES; ++i) mbar_init(&full[0][0] + i, 1);
        fence_mbar_init();
        prefetch_tmap(&map);
    }
    if (tid < W * 2) parts[tid >> 1][tid & 1].unit = -1;
    // What ran before is complete. (No read-only loads below: they may move across this, and what it
    // waits for may write the queries, tables and lengths.)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    PagedSplit sp{};
    PagedUnit only{};                                        // alone: the CTA's unit
    long long c_begin;
    int c_blocks;                                            // at most 2^28 (64 layers, 8 heads, 2^30 rows over 148 ranges)
    if (alone) {
        const int i = c / alone, rank = c - i * alone;       // the CTA's unit, and its place in the cluster
        only = paged_unit_alone(i, a.n, hkv, ((a.cols << a.kv.shift) + BLK - 1) / BLK);
        const int given = a.lengths[only.b], len = paged_length(given, a.cols, a.kv.shift);
        if (given != len && tid == 0) atomicCAS(a.error + ERR_DATA, 0, PAGED_BAD_LENGTH);
        only.nblk = (len + BLK - 1) / BLK;
        if (len == 0) {                                      // (for the whole cluster)
            for (int col = tid; rank == 0 && col < GROUP * D; col += T) a.out[(size_t)i * GROUP * D + col] = 0.f;
            return;
        }
        const int from = only.nblk * rank / alone;
        c_begin = only.off + from;
        c_blocks = only.nblk * (rank + 1) / alone - from;
        __syncthreads();                                     // the barriers and parts above are ready
    } else {
        sp = scan_lengths(a, start, warp_sum);               // (its barriers cover them too)
        if (sp.total == 0 || c >= sp.ctas) {
            if (tid < 2) shared_of(a)[c * 2 + tid].nrec = 0;
            return;
        }
        if (tid < 2) shared_of(a)[c * 2 + tid].nrec = 0;     // until the merge finds a shared unit
        c_begin = sp.begin(c);
        c_blocks = (int)(sp.begin(c + 1) - c_begin);
    }
    auto unit_of = [&](long long g) { return alone ? only : paged_unit_of(start, a.n, hkv, g); };
    // this warp's blocks [g_begin, g_end) of the range
    const long long g_begin = c_begin + c_blocks * warp / W, g_end = c_begin + c_blocks * (warp + 1) / W;
    const float qscale = 1.4426950408889634f * 0.08838834764831845f;   // log2(e)/sqrt(128)
    const int mask = (1 << a.kv.shift) - 1;
    uint8_t* const my_ring = ring + warp * (STAGES * STAGE);
    uint64_t* const my_full = full[warp];
    uint32_t issued = 0, consumed = 0;

    if (g_begin < g_end) {
        // ---- producer side: 32 blocks are looked up at a time, one a lane, a batch ahead ----
        PagedUnit u = unit_of(min(g_begin + lane, g_end - 1));
        // queries: lane's 8 channels of head lane / 16, loaded a unit ahead
        float4 q_raw[2];
        auto load_q = [&](const PagedUnit& w) {
            const float* row = a.q + ((((size_t)w.l * a.n + w.b) * hkv + w.kh) * GROUP) * D + lane * 8;
            q_raw[0] = reinterpret_cast<const float4*>(row)[0];
            q_raw[1] = reinterpret_cast<const float4*>(row)[1];
        };
        int page_next = -1, place_next = 0;                  // next batch: page id, first row within the page's K rows of the head
        auto look_up = [&](const PagedUnit& w, long long g) {
            const int t0 = (int)(g - w.off) * BLK;
            page_next = a.table[(size_t)w.b * a.cols + (t0 >> a.kv.shift)];
            place_next = (((a.layer0 + w.l) * 2 * hkv + w.kh) << a.kv.shift) + (t0 & mask);
        };
        // row of the block's K in the pool's matrix of planes ((page, layer), K|V, head); -1: no such page
        auto place = [&]() { return a.kv.has(page_next) ? ((page_next * a.kv.layers * 2 * hkv) << a.kv.shift) + place_next : -1; };
        look_up(u, min(g_begin + lane, g_end - 1));
        auto from_first = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
        u.l = from_first(u.l); u.b = from_first(u.b); u.kh = from_first(u.kh); u.nblk = from_first(u.nblk);
        u.off = __shfl_sync(0xffffffffu, u.off, 0);          // the unit of g_begin
        load_q(u);                                           // (before the copies: it would queue behind them)
        const uint64_t once = policy_evict_first();
        int rows_now = place();                              // of the batch being copied
        const int n_blocks = (int)(g_end - g_begin);
        uint32_t valid = 0;                                  // bit per stage: the block was copied
        auto produce = [&]() {
            if ((int)issued >= n_blocks) return;
            if ((issued & 31) == 0) {
                if (issued) rows_now = place();
                const long long next = g_begin + issued + 32 + lane;
                if (next - lane < g_end) look_up(unit_of(min(next, g_end - 1)), min(next, g_end - 1));
            }
            const int stage = issued % STAGES, row = __shfl_sync(0xffffffffu, rows_now, issued & 31);
            const bool ok = row >= 0;
            valid = ok ? valid | 1u << stage : valid & ~(1u << stage);
            if (lane == 0) {
                if (ok) mbar_arrive_expect_tx(&my_full[stage], STAGE);
                else { mbar_arrive(&my_full[stage]); atomicCAS(a.error + ERR_DATA, 0, PAGED_BAD_PAGE); }
            }
            __syncwarp();
            if (ok && lane < 4) {                            // lane: K or V, channel half
                const int kv = lane >> 1, half = lane & 1;
                tma_load_2d_once(my_ring + stage * STAGE + kv * HALF_STAGE + half * (HALF_STAGE / 2), &map, half * 64,
                            row + (kv * hkv << a.kv.shift), &my_full[stage], once);
            }
            ++issued;
        };
        for (int i = 0; i < STAGES; ++i) produce();

        // shared-memory rows this lane names to ldmatrix (16-byte chunk x of row r sits at chunk
        // x ^ (r % 8) of its 128-byte line); K: rows in the low bit of the matrix index, V: chunks
        const int mi = lane >> 3, k_row = (lane & 7) + (mi & 1) * 8, v_row = (lane & 7) + (mi >> 1) * 8;
        const uint32_t ring_addr = smem_u32(my_ring);
        // a unit's query halves, packed (high, low), go through the slot of the warp's last part, which
        // is written after that part's queries are in registers
        uint32_t* const s_q = reinterpret_cast<uint32_t*>(s_part[warp][1]);
        for (long long g = g_begin; g < g_end;) {
            const int cnt = (int)(min(u.off + u.nblk, g_end) - g), blk0 = (int)(g - u.off);
            const int len = row_length(a, u.b);
            uint32_t qf[16];                                 // column g8: head (g8 / 2) % 2, its high or low half by g8 % 2
            float unscale;                                   // logit = unscale * dot product, of head `head`
            {
                float v[8] = {q_raw[0].x, q_raw[0].y, q_raw[0].z, q_raw[0].w, q_raw[1].x, q_raw[1].y, q_raw[1].z, q_raw[1].w};
                float top = 0.f;
                #pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
                #pragma unroll
                for (int o = 1; o <= 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                // scale = 2^(13 - exponent of top), at most 2^100
                const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -87), 127);
                const float scale = __uint_as_float((uint32_t)(13 - e + 127) << 23);
                unscale = __shfl_sync(0xffffffffu, qscale * __uint_as_float((uint32_t)(e - 13 + 127) << 23), head * 16);
                uint32_t h[8];
                #pragma unroll
                for (int i = 0; i < 8; ++i) h[i] = split_half(v[i] * scale);
                uint4* to = reinterpret_cast<uint4*>(s_q + lane * 8);
                to[0] = make_uint4(h[0], h[1], h[2], h[3]);
                to[1] = make_uint4(h[4], h[5], h[6], h[7]);
                __syncwarp();
                // channels 16 k + 2 j4 + {0, 1} and + {8, 9} of step k
                const uint2* from = reinterpret_cast<const uint2*>(s_q + (g8 >> 1 & 1) * D + 2 * j4);
                #pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint2 x = from[4 * i];
                    qf[i] = __byte_perm(x.x, x.y, g8 & 1 ? 0x7632 : 0x5410);
                }
                __syncwarp();
            }
            PagedUnit nu = u;                                // the next unit's queries, loaded meanwhile
            if (g + cnt < g_end) {
                paged_next_unit(start, a.n, hkv, nu);
                load_q(nu);
            }
            float m = -INFINITY, l = 0.f;                    // of head `head`: maximum - 14, this lane's share of the sum
            float acc[8][4];                                 // [16-channel tile]: channels g8, g8 + 8; high and low columns of `head`
            #pragma unroll
            for (int i = 0; i < 8; ++i)
                #pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
            for (int j = 0; j < cnt; ++j) {
                const int stage = consumed % STAGES;
                bool got = mbar_wait(&my_full[stage], (consumed / STAGES) & 1, &abort_flag);
                if (!got) { abort_flag = 1; atomicCAS(a.error, 0, WAIT_CODE); }
                got = __all_sync(0xffffffffu, got);
                const int rows = min(BLK, len - (blk0 + j) * BLK);
                if (got && (valid >> stage & 1)) {
                    const uint32_t k_addr = ring_addr + stage * STAGE + k_row * 128, v_addr = ring_addr + stage * STAGE + HALF_STAGE + v_row * 128;
                    // logits: rows g8 and g8 + 8 of the block, columns 2 j4 (high) and 2 j4 + 1 (low)
                    float sc[4][4];
                    #pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint32_t kf[4];
                        const int chunk = (2 * k + (mi >> 1)) & 7;
                        ldmatrix4(kf, k_addr + (k >> 2) * (HALF_STAGE / 2) + ((chunk ^ (k_row & 7)) << 4));
                        if (k < 4) mma16816_new(sc[k], kf, qf[2 * k], qf[2 * k + 1]);
                        else mma16816(sc[k - 4], kf, qf[2 * k], qf[2 * k + 1]);
                    }
                    float s0 = (((sc[0][0] + sc[1][0]) + (sc[2][0] + sc[3][0])) + ((sc[0][1] + sc[1][1]) + (sc[2][1] + sc[3][1]))) * unscale;
                    float s1 = (((sc[0][2] + sc[1][2]) + (sc[2][2] + sc[3][2])) + ((sc[0][3] + sc[1][3]) + (sc[2][3] + sc[3][3]))) * unscale;
                    if (rows < BLK) {
                        // rows past the length: no logit, and zero V rows, whatever their page holds
                        if (g8 >= rows) s0 = -INFINITY;
                        if (g8 + 8 >= rows) s1 = -INFINITY;
                        for (int i = rows * 8 + lane; i < BLK * 8; i += 32) {
                            uint4* v = reinterpret_cast<uint4*>(my_ring + stage * STAGE + HALF_STAGE) + i;
                            v[0] = make_uint4(0, 0, 0, 0);
                            v[BLK * 8] = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_smem();            // before the stage's next copy
                        __syncwarp();
                    }
                    if (WEIGHTS && j4 < GROUP) {
                        float* to = a.logits + (g + j) * (BLK * 2) + g8 * 2 + j4;
                        to[0] = s0;
                        to[16] = s1;
                    }
                    float mb = fmaxf(s0, s1);
                    #pragma unroll
                    for (int o = 4; o <= 16; o <<= 1) mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, o));
                    mb -= 14.f;
                    if (__any_sync(0xffffffffu, mb > m)) {
                        const float mn = fmaxf(m, mb), scale = exp2_from(m, mn);
                        m = mn;
                        l *= scale;
                        #pragma unroll
                        for (int i = 0; i < 8; ++i)
                            #pragma unroll
                            for (int e = 0; e < 4; ++e) acc[i][e] *= scale;
                    }
                    // weights of the block's own maximum, whose halves therefore hold them, and the block's factor
                    const float p0 = g8 < rows ? exp2_from(s0, mb) : 0.f, p1 = g8 + 8 < rows ? exp2_from(s1, mb) : 0.f;
                    const float factor = exp2_from(mb, m);
                    l += factor * (p0 + p1);
                    // this lane's operand: rows 2 j4 + {0, 1, 8, 9} of column g8 (head (g8 / 2) % 2, half g8 % 2)
                    const uint32_t h0 = split_half(p0), h1 = split_half(p1);
                    const int from = 8 * j4 + (g8 >> 1 & 1);
                    const uint32_t x0 = __shfl_sync(0xffffffffu, h0, from), x1 = __shfl_sync(0xffffffffu, h0, from + 4);
                    const uint32_t x2 = __shfl_sync(0xffffffffu, h1, from), x3 = __shfl_sync(0xffffffffu, h1, from + 4);
                    const uint32_t pick = g8 & 1 ? 0x7632 : 0x5410;
                    const uint32_t b0 = __byte_perm(x0, x1, pick), b1 = __byte_perm(x2, x3, pick);
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint32_t vf[4];
                        const int chunk = (2 * i + (mi & 1)) & 7;
                        ldmatrix4_trans(vf, v_addr + (i >> 2) * (HALF_STAGE / 2) + ((chunk ^ (v_row & 7)) << 4));
                        float pv[4];
                        mma16816_new(pv, vf, b0, b1);
                        #pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][e] += factor * pv[e];
                    }
                }
                __syncwarp();                                // the stage is read by all lanes
                if (got) {
                    ++consumed;
                    produce();
                }
            }
            // ---- the unit's part is done: column `head`; lanes j4 < 2 write channels g8, the others g8 + 8 ----
            #pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const int unit = (u.l * a.n + u.b) * hkv + u.kh;
            const bool whole = cnt == u.nblk;
            float* to = a.out + (size_t)unit * GROUP * D;
            if (!whole) {
                const int slot = g == g_begin ? 0 : 1;       // (a middle unit is whole)
                to = s_part[warp][slot];
                if (lane == 0) {
                    Part& p = parts[warp][slot];
                    p.unit = unit; p.blk0 = blk0; p.cnt = cnt; p.nblk = u.nblk; p.g = g;
                }
                if (lane < GROUP) { parts[warp][slot].m[lane] = m; parts[warp][slot].l[lane] = l; }
            }
            const float inv = whole ? 1.f / l : 1.f;
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = (j4 < 2 ? acc[i][0] + acc[i][1] : acc[i][2] + acc[i][3]);
                to[head * D + 16 * i + g8 + (j4 < 2 ? 0 : 8)] = x * inv;
            }
            if (WEIGHTS && whole) {
                const float M[GROUP] = {__shfl_sync(0xffffffffu, m, 0), __shfl_sync(0xffffffffu, m, 1)};
                const float L[GROUP] = {__shfl_sync(0xffffffffu, l, 0), __shfl_sync(0xffffffffu, l, 1)};
                __syncwarp();                                // the warp's own logits
                add_weights(a, u.l, u.b, u.kh, len, 0, cnt, g, M, L, lane, 32);
            }
            g += cnt;
            u = nu;
        }
        // drain: copies issued but not consumed (after an expired wait) must land before the CTA exits
        for (; consumed < issued; ++consumed) mbar_wait(&my_full[consumed % STAGES], (consumed / STAGES) & 1, &never_abort, 500000000ull);
    }
    __syncthreads();

    // ---- merge the warps' parts: those of one unit are neighbours in the order of the blocks ----
    // A single unit by all threads, a column or two each; several by a warp each (64 ragged rows 95.5 -> 94.2 us,
    // 33 of up to 512 17.9 -> 16.3 us against one after the other; a single unit is 0.3 us faster by all).
    // Every warp holds all parts, two lanes each: lane is part lane % 16 and head lane / 16.
    static_assert(W * 2 <= 16 && GROUP * D % T == 0, "two heads of all parts fit a warp; whole rounds of columns");
    const int part = lane & 15, part_head = lane >> 4;
    Part p{};
    p.unit = -1;
    if (part < W * 2) p = parts[part >> 1][part & 1];
    const float p_m = part_head ? p.m[1] : p.m[0], p_l = part_head ? p.l[1] : p.l[0];
    const unsigned all = __ballot_sync(0xffffffffu, p.unit >= 0) & 0xffff;
    bool single = true;
    int turn = 0;                                            // units so far
    for (unsigned left = all; left; ++turn) {
        const int first = __ffs(left) - 1;
        const int unit = __shfl_sync(0xffffffffu, p.unit, first);
        const bool mine = p.unit == unit;
        const unsigned group = __ballot_sync(0xffffffffu, mine) & 0xffff;
        left &= ~group;
        single = group == all;
        if (!single && turn % W != warp) continue;
        const int blk0 = __shfl_sync(0xffffffffu, p.blk0, first), nblk = __shfl_sync(0xffffffffu, p.nblk, first);
        const long long g = __shfl_sync(0xffffffffu, p.g, first);
        const int cnt = __reduce_add_sync(0xffffffffu, mine && part_head == 0 ? p.cnt : 0);
        float top = mine ? p_m : -INFINITY;
        #pragma unroll
        for (int x = 8; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float f = mine ? exp2_from(p_m, top) : 0.f;
        float sum = mine ? f * p_l : 0.f;
        #pragma unroll
        for (int x = 8; x >= 1; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const float M[GROUP] = {__shfl_sync(0xffffffffu, top, 0), __shfl_sync(0xffffffffu, top, 16)};
        const float L[GROUP] = {__shfl_sync(0xffffffffu, sum, 0), __shfl_sync(0xffffffffu, sum, 16)};
        const int slot = g != c_begin;
        float* rec = a.records + ((size_t)c * 2 + slot) * PARTIAL_FLOATS;
        if (single) {
            constexpr int COLS = GROUP * D / T;              // of a thread, T apart
            float o[COLS];
            #pragma unroll
            for (int x = 0; x < COLS; ++x) {
                const int col = x * T + tid;
                o[x] = 0.f;
                #pragma unroll
                for (int k = 0; k < W * 2; ++k) {
                    const float fk = __shfl_sync(0xffffffffu, f, k + (col >= D ? 16 : 0));   // (a warp's columns are of one head)
                    if (group >> k & 1) o[x] += fk * s_part[k >> 1][k & 1][col];
                }
            }
            if (cnt == nblk) {
                #pragma unroll
                for (int x = 0; x < COLS; ++x)
                    a.out[(size_t)unit * GROUP * D + x * T + tid] = o[x] / (x * T + tid >= D ? L[1] : L[0]);
                if (WEIGHTS) {
                    const int lb = unit / hkv, row_l = lb / a.n, row_b = lb - row_l * a.n, row_kh = unit - lb * hkv;
                    add_weights(a, row_l, row_b, row_kh, row_length(a, row_b), 0, cnt, g, M, L, tid, T);
                }
            } else if (alone) {
                #pragma unroll
                for (int x = 0; x < COLS; ++x) joint.o[x * T + tid] = o[x];
                if (tid < GROUP) { joint.m[tid] = tid ? M[1] : M[0]; joint.l[tid] = tid ? L[1] : L[0]; }
                if (tid == 0) joint.cnt = cnt;
            } else {
                #pragma unroll
                for (int x = 0; x < COLS; ++x) rec[4 + x * T + tid] = o[x];
            }
        } else if (W == WARPS) {
            float4 o[GROUP];                                 // channels 4 lane to 4 lane + 3 of both heads
            #pragma unroll
            for (int k = 0; k < GROUP; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (unsigned parts_left = group; parts_left; parts_left &= parts_left - 1) {
                const int i = __ffs(parts_left) - 1;
                #pragma unroll
                for (int k = 0; k < GROUP; ++k) {
                    const float fk = __shfl_sync(0xffffffffu, f, i + 16 * k);
                    const float4 x = reinterpret_cast<const float4*>(s_part[i >> 1][i & 1] + k * D)[lane];
                    o[k].x += fk * x.x; o[k].y += fk * x.y; o[k].z += fk * x.z; o[k].w += fk * x.w;
                }
            }
            const bool whole = cnt == nblk;
            if (WEIGHTS && lane == 0) {
                Whole& w = wholes[turn];
                w.unit = unit; w.cnt = whole ? cnt : 0; w.g = g;
                w.m[0] = M[0]; w.m[1] = M[1]; w.l[0] = L[0]; w.l[1] = L[1];
            }
            #pragma unroll
            for (int k = 0; k < GROUP; ++k) {
                if (whole)
                    reinterpret_cast<float4*>(a.out + ((size_t)unit * GROUP + k) * D)[lane] =
                        make_float4(o[k].x / L[k], o[k].y / L[k], o[k].z / L[k], o[k].w / L[k]);
                else
                    reinterpret_cast<float4*>(rec + 4 + k * D)[lane] = o[k];
            }
        }
        if (!alone && cnt != nblk && lane == 0 && (!single || warp == 0)) {
            *reinterpret_cast<float4*>(rec) = make_float4(M[0], M[1], L[0], L[1]);
            const long long off = g - blk0;
            Shared s;
            s.first = sp.range_of(off);
            s.nrec = sp.range_of(off + nblk - 1) - s.first + 1;
            s.first_slot = off != sp.begin(s.first);
            s.unit = unit; s.blk0 = blk0; s.cnt = cnt; s.g = g;
            shared_of(a)[c * 2 + slot] = s;
        }
    }
    if (WEIGHTS && !single) {
        __syncthreads();
        for (int e = 0; e < turn; ++e) {
            const Whole w = wholes[e];
            const bool by_all = w.cnt > 4 * W;               // those of a short unit by one warp
            if (w.cnt == 0 || !(by_all || warp == e % W)) continue;
            const int lb = w.unit / hkv, row_l = lb / a.n, row_b = lb - row_l * a.n, row_kh = w.unit - lb * hkv;
            add_weights(a, row_l, row_b, row_kh, row_length(a, row_b), 0, w.cnt, w.g, w.m, w.l, by_all ? tid : lane, by_all ? T : 32);
        }
    }
    if (alone <= 1) return;
    // ---- join the cluster's parts (none where one CTA held the whole unit) ----
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    int cnts[4], total = 0;
    float M[GROUP] = {-INFINITY, -INFINITY}, L[GROUP] = {0.f, 0.f}, f[4][GROUP];
    #pragma unroll
    for (int r = 0; r < 4; ++r) {
        cnts[r] = 0;
        f[r][0] = f[r][1] = -INFINITY;
        if (r >= alone) continue;
        const Joint* x = cluster.map_shared_rank(&joint, r);
        cnts[r] = x->cnt;
        f[r][0] = x->m[0]; f[r][1] = x->m[1];
        total += cnts[r];
    }
    if (total == only.nblk) {
        #pragma unroll
        for (int r = 0; r < 4; ++r)
            #pragma unroll
            for (int k = 0; k < GROUP; ++k)
                if (cnts[r]) M[k] = fmaxf(M[k], f[r][k]);
        float sum = 0.f;
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (!cnts[r]) continue;
            const Joint* x = cluster.map_shared_rank(&joint, r);
            #pragma unroll
            for (int k = 0; k < GROUP; ++k) {
                f[r][k] = exp2_from(f[r][k], M[k]);
                L[k] += f[r][k] * x->l[k];
            }
            sum += (tid < D ? f[r][0] : f[r][1]) * x->o[tid];
        }
        const int i = c / alone;
        if (c - i * alone == 0) a.out[(size_t)i * GROUP * D + tid] = sum / (tid < D ? L[0] : L[1]);
        if (WEIGHTS && c_blocks)
            add_weights(a, only.l, only.b, only.kh, row_length(a, only.b), (int)(c_begin - only.off), c_blocks, c_begin, M, L, tid, THREADS);
    }
    cluster.sync();                                          // until the others have read this CTA's memory
}

// CTA (range c, side): if c is the first range of the side's shared unit, joins the unit; with weights,
// adds those of the range's part of it, shared with JOIN_PARTS - 1 more CTAs (2 rows of 131071 and
// 77777: 162.5 -> 158.2 us; no slower where there is little to add). Beside that, before the first
// launch is done: rows of length 0. (One CTA per side rather than one after the other: the chain of
// latencies is short.)
__global__ void __launch_bounds__(JOIN_THREADS, 5) attn_paged_join_kernel(const PagedAttnArgs a) {
    __shared__ float s_f[CTAS][GROUP];                       // factor of each record
    __shared__ float red[2 * GROUP][JOIN_THREADS / 32];
    __shared__ __align__(16) float s_sum[JOIN_GROUPS][GROUP * D];
    static_assert(CTAS <= JOIN_THREADS && GROUP * D == JOIN_THREADS, "one record, and one column, a thread");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x >> 1;
    const int part = blockIdx.y;
    const int row_floats = GROUP * a.kv.hkv * D;
    for (int b = tid; b < a.n && blockIdx.x + part == 0; b += JOIN_THREADS)
        if (a.lengths[b] != row_length(a, b)) atomicCAS(a.error + ERR_DATA, 0, PAGED_BAD_LENGTH);
    for (int i = blockIdx.x; part == 0 && i < a.n_layers * a.n; i += gridDim.x)
        if (row_length(a, i % a.n) == 0)
            for (int j = tid * 4; j < row_floats; j += JOIN_THREADS * 4)
                *reinterpret_cast<float4*>(a.out + (size_t)i * row_floats + j) = make_float4(0.f, 0.f, 0.f, 0.f);
    asm volatile("griddepcontrol.wait;" ::: "memory");       // the split launch is complete and its stores visible
    const Shared s = shared_of(a)[blockIdx.x];
    if (s.nrec == 0 || (s.first != c && !a.add_weights)) return;
    // record i of the unit: range first + i, slot 0 but in the first range
    const float* first = a.records + ((size_t)s.first * 2 + s.first_slot) * PARTIAL_FLOATS;
    const float* others = a.records + (size_t)s.first * 2 * PARTIAL_FLOATS;
    float M[GROUP] = {-INFINITY, -INFINITY}, L[GROUP] = {0.f, 0.f};
    float4 st = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
    if (tid < s.nrec) st = *reinterpret_cast<const float4*>(tid ? others + (size_t)tid * 2 * PARTIAL_FLOATS : first);
    M[0] = st.x; M[1] = st.y;
    #pragma unroll
    for (int k = 0; k < GROUP; ++k) {
        #pragma unroll
        for (int x = 16; x >= 1; x >>= 1) M[k] = fmaxf(M[k], __shfl_xor_sync(0xffffffffu, M[k], x));
    }
    if (lane < GROUP) red[lane][warp] = lane ? M[1] : M[0];
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < GROUP; ++k)
        #pragma unroll
        for (int w = 0; w < JOIN_THREADS / 32; ++w) M[k] = fmaxf(M[k], red[k][w]);
    if (tid < s.nrec) {
        const float f0 = exp2_from(st.x, M[0]), f1 = exp2_from(st.y, M[1]);
        s_f[tid][0] = f0; s_f[tid][1] = f1;
        L[0] = f0 * st.z; L[1] = f1 * st.w;
    }
    #pragma unroll
    for (int k = 0; k < GROUP; ++k) {
        #pragma unroll
        for (int x = 16; x >= 1; x >>= 1) L[k] += __shfl_xor_sync(0xffffffffu, L[k], x);
    }
    if (lane < GROUP) red[GROUP + lane][warp] = lane ? L[1] : L[0];
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < GROUP; ++k) {
        L[k] = 0.f;
        #pragma unroll
        for (int w = 0; w < JOIN_THREADS / 32; ++w) L[k] += red[GROUP + k][w];
    }
    if (s.first == c && part == 0) {
        // four columns a thread, every fourth record a group, then the groups in order
        const int grp = tid / (GROUP * D / 4), col = tid % (GROUP * D / 4) * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll 4
        for (int i = grp; i < s.nrec; i += JOIN_GROUPS) {
            const float4 x = *reinterpret_cast<const float4*>((i ? others + (size_t)i * 2 * PARTIAL_FLOATS : first) + 4 + col);
            const float f = s_f[i][col >= D];
            o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
        }
        *reinterpret_cast<float4*>(&s_sum[grp][col]) = o;
        __syncthreads();
        float sum = 0.f;
        #pragma unroll
        for (int k = 0; k < JOIN_GROUPS; ++k) sum += s_sum[k][tid];
        a.out[(size_t)s.unit * GROUP * D + tid] = sum / (tid < D ? L[0] : L[1]);
    }
    if (a.add_weights) {
        const int lb = s.unit / a.kv.hkv, b = lb % a.n;
        add_weights(a, lb / a.n, b, s.unit % a.kv.hkv, row_length(a, b), s.blk0, s.cnt, s.g, M, L, part * JOIN_THREADS + tid,
                    JOIN_PARTS * JOIN_THREADS);
    }
}

}  // namespace

// Workspace: [records][shared][logits].
static constexpr size_t RECORD_BYTES = (size_t)CTAS * 2 * PARTIAL_FLOATS * sizeof(float);
static constexpr size_t SHARED_BYTES = (size_t)CTAS * 2 * sizeof(Shared);
static_assert(RECORD_BYTES % 16 == 0 && SHARED_BYTES % 16 == 0, "each part 16-byte aligned");

size_t paged_attn_workspace(int n, int n_layers, int hkv, int max_rows, bool weights) {
    const size_t blocks = (size_t)n * n_layers * hkv * ((max_rows + BLK - 1) / BLK);
    return RECORD_BYTES + SHARED_BYTES + (weights ? blocks * BLK * 2 * sizeof(float) : 0);
}

// With `overlap` the CTAs may start while the launch before this one ends; they wait for its end themselves.
template <class... Params, class... Args>
static cudaError_t launch(void (*kernel)(Params...), bool overlap, dim3 ctas, int cluster, int threads, size_t smem, cudaStream_t s,
                          const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = ctas; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlap;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <bool WEIGHTS, int W>
static cudaError_t launch_split(const PagedAttnArgs& a, const CUtensorMap& map, int ctas, cudaStream_t s) {
    const auto kernel = attn_paged_split_kernel<WEIGHTS, W>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_bytes(W));
    return e != cudaSuccess ? e : launch(kernel, a.overlap, ctas, a.alone > 1 ? a.alone : 1, W * 32, ring_bytes(W), s, a, map);
}

cudaError_t launch_paged_attn(PagedAttnArgs a, const CUtensorMap& map, void* workspace, cudaStream_t s) {
    char* ws = static_cast<char*>(workspace);
    a.records = reinterpret_cast<float*>(ws);
    a.shared = ws + RECORD_BYTES;
    a.logits = reinterpret_cast<float*>(ws + RECORD_BYTES + SHARED_BYTES);
    const long long units = (long long)a.n * a.n_layers * a.kv.hkv;
    const int most = ((a.cols << a.kv.shift) + BLK - 1) / BLK;
    int warps = WARPS;
    if (a.n > 1) a.alone = paged_ctas_alone(units, most, CTAS, WARPS);
    else {
        const PagedAlone p = paged_alone_equal(units, most, CTAS, WARPS);
        a.alone = p.ctas;
        warps = p.warps;
    }
    const int ctas = a.alone ? (int)units * a.alone : CTAS;
    const cudaError_t e = warps == WARPS ? a.add_weights ? launch_split<true, WARPS>(a, map, ctas, s) : launch_split<false, WARPS>(a, map, ctas, s)
                                         : a.add_weights ? launch_split<true, WARPS / 2>(a, map, ctas, s) : launch_split<false, WARPS / 2>(a, map, ctas, s);
    return e != cudaSuccess || a.alone ? e : launch(attn_paged_join_kernel, true, dim3(CTAS * 2, a.add_weights ? JOIN_PARTS : 1), 1, JOIN_THREADS, 0, s, a);
}

}  // namespace qattn
