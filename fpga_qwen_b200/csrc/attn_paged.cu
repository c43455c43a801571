// attn_paged.cu — decode attention of one query row per sequence over a paged KV cache.
//
// For row b with L = lengths[b] cached rows, layer l and KV head kh, both query heads h of the
// group: s_t = q_h . k_t / sqrt(128), p = softmax(s), out_h = sum_t p_t v_t, all in FP32 over the
// FP16 rows; with add_weights also weights[t] += p_t of both heads.
//
// Bound by HBM: 512 bytes of K and V a row and KV head for 1,024 flops. What keeps HBM busy:
//   * Even split (stream-K style). The 16-row blocks of all (layer, row, KV head) units are laid
//     end to end and cut into equal ranges, one per CTA (2 per SM), whatever the lengths are;
//     lengths are read on the device, so every CTA first scans them. A range can end inside one
//     unit and continue in the next.
//   * Every warp is its own pipeline: it takes every fourth block of the range, and one lane keeps
//     STAGES blocks (K and V rows, 8 KB) in flight into the warp's ring with bulk copies, across
//     unit boundaries, 192 KB per SM. A block never crosses a page, so a block is one page id; the
//     next id is loaded one block ahead. No barrier between the warps inside a unit: each has its
//     own running maximum and sum, merged through shared memory when the unit's part ends.
//   * Both query heads of a KV head share its rows in registers.
// A unit inside one range is finished there; a unit that several ranges share leaves one record
// (max, sum, 2 x 128 partial output) per range, and a second launch, whose CTAs wait ready behind
// the first's (programmatic dependent launch), joins them in range order: no atomics, so the
// result does not depend on timing. At most two units of a range are shared (its first and its
// last), so the records are 2 per CTA, whatever the batch.
//
// The weights need the final maximum and sum: the logits go to the workspace (8 bytes a row and
// KV head against 512 of K and V) and become weights when the unit is finished, in this launch or
// in the joining one. Each (row, KV head) weight gets one FP32 addition.
//
// Every wait is bounded: on expiry the CTA records an error code, consumes no further block, and
// drains its copies before it exits.
#include "qattn_common.cuh"
#include "sm100.cuh"

namespace qattn {
namespace {

using namespace sm100;

constexpr int THREADS = 128, WARPS = THREADS / 32;
constexpr int BLK = PAGED_BLK;
constexpr int STAGES = 3;                     // blocks in flight per warp
constexpr int HALF_STAGE = BLK * D * 2;       // K rows, then V rows of a block: 4 KB each
constexpr int STAGE = 2 * HALF_STAGE;
constexpr int RING = WARPS * STAGES * STAGE;
constexpr int WAIT_CODE = 43;                 // error code of an expired wait
constexpr int CTAS = NUM_SMS_B200 * 2;        // ranges
constexpr int MIN_BLOCKS = 4;                 // blocks per range, at least (64 rows)

__device__ __forceinline__ int row_length(const PagedAttnArgs& a, int b) {
    return paged_length(a.lengths[b], a.cols, a.kv.shift);
}

// start[b] = blocks of rows [0, b); called by all threads of the CTA, n <= MAX_PAGED_BATCH.
__device__ PagedSplit scan_lengths(const PagedAttnArgs& a, int* start, int* warp_sum) {
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
    for (int w = 0; w < warp; ++w) base += warp_sum[w];
    #pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = tid * PER + i;
        if (b < a.n) start[b] = base + v[i];
    }
    if (tid == THREADS - 1) start[a.n] = base + sum;
    __syncthreads();
    return paged_split((long long)a.n_layers * a.kv.hkv * start[a.n], CTAS, MIN_BLOCKS);
}

__device__ __forceinline__ void unpack8(const uint4 u, float f[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    #pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 t = __half22float2(h[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
}

// exp2(x - m) where m is a maximum that may still be -inf (nothing seen, or only -inf logits).
__device__ __forceinline__ float exp2_from(float x, float m) { return exp2f(x - (m == -INFINITY ? 0.f : m)); }

// weights += p for the rows of blocks [g, g + cnt) of unit u, by all threads of the CTA.
__device__ __forceinline__ void add_weights(const PagedAttnArgs& a, const PagedUnit& u, long long g, int cnt, const float M[2],
                                            const float L[2]) {
    const int t0 = (int)(g - u.off) * BLK, len = row_length(a, u.b);
    const int t1 = min(t0 + cnt * BLK, len);
    const float* s = a.logits + g * (BLK * 2);
    for (int t = t0 + (int)threadIdx.x; t < t1; t += THREADS) {
        const float2 x = *reinterpret_cast<const float2*>(s + (size_t)(t - t0) * 2);
        const int page = a.table[(size_t)u.b * a.cols + (t >> a.kv.shift)];
        if (a.kv.has(page))
            atomicAdd(a.kv.weight(page, a.layer0 + u.l, u.kh, t & ((1 << a.kv.shift) - 1)),
                      exp2_from(x.x, M[0]) / L[0] + exp2_from(x.y, M[1]) / L[1]);
    }
}

__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) {
    unsigned long long r, ua = *reinterpret_cast<unsigned long long*>(&a), ub = *reinterpret_cast<unsigned long long*>(&b),
                          uc = *reinterpret_cast<unsigned long long*>(&c);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(ua), "l"(ub), "l"(uc));
    return *reinterpret_cast<float2*>(&r);
}

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// v[i] summed over the 16 lanes of each half-warp, for i = 0..15: the lane with sl == i gets sum i.
__device__ __forceinline__ float transpose_sum16(const float (&v)[16], int sl) {
    float w8[8], w4[4], w2[2];
    #pragma unroll
    for (int i = 0; i < 8; ++i) w8[i] = (sl & 8 ? v[i + 8] : v[i]) + __shfl_xor_sync(0xffffffffu, sl & 8 ? v[i] : v[i + 8], 8);
    #pragma unroll
    for (int i = 0; i < 4; ++i) w4[i] = (sl & 4 ? w8[i + 4] : w8[i]) + __shfl_xor_sync(0xffffffffu, sl & 4 ? w8[i] : w8[i + 4], 4);
    #pragma unroll
    for (int i = 0; i < 2; ++i) w2[i] = (sl & 2 ? w4[i + 2] : w4[i]) + __shfl_xor_sync(0xffffffffu, sl & 2 ? w4[i] : w4[i + 2], 2);
    return (sl & 1 ? w2[1] : w2[0]) + __shfl_xor_sync(0xffffffffu, sl & 1 ? w2[0] : w2[1], 1);
}

__global__ void __launch_bounds__(THREADS, 2) attn_paged_split_kernel(const PagedAttnArgs a) {
    extern __shared__ __align__(128) uint8_t ring[];         // [WARPS][STAGES][K rows | V rows]
    __shared__ __align__(8) uint64_t full[WARPS][STAGES];
    __shared__ int start[MAX_PAGED_BATCH + 1];
    __shared__ int warp_sum[WARPS];
    __shared__ float s_stat[2][WARPS][4];                    // by segment parity: max and sum of both heads
    __shared__ __align__(16) float s_acc[2][WARPS][GROUP][D];
    __shared__ int abort_flag, never_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hw = lane >> 4, sl = lane & 15;                // half-warp: rows of one parity; 8 channels a lane
    const int hq = GROUP * a.kv.hkv;
    if (tid == 0) {
        abort_flag = 0; never_abort = 0;
        for (int i = 0; i < WARPS * STAGES; ++i) mbar_init(&full[0][0] + i, 1);
        fence_mbar_init();
    }
    const PagedSplit sp = scan_lengths(a, start, warp_sum);   // its barriers publish the ring's too
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x == 0)
        for (int b = tid; b < a.n; b += THREADS)
            if (a.lengths[b] != row_length(a, b)) atomicCAS(a.error, 0, PAGED_BAD_LENGTH);
    // rows without keys: zeros
    for (int i = blockIdx.x; i < a.n_layers * a.n; i += gridDim.x) {
        const int b = i % a.n;
        if (start[b + 1] == start[b])
            for (int j = tid; j < hq * D; j += THREADS) a.out[(size_t)i * hq * D + j] = 0.f;
    }
    const int c = blockIdx.x;
    if (sp.total == 0 || c >= sp.ctas) return;
    const long long g_begin = sp.begin(c), g_end = sp.begin(c + 1);
    const float qscale = 1.4426950408889634f * 0.08838834764831845f;   // log2(e)/sqrt(128)
    const int mask = (1 << a.kv.shift) - 1;
    uint8_t* const my_ring = ring + warp * (STAGES * STAGE);
    uint64_t* const my_full = full[warp];

    // ---- producer side of the warp: blocks g_begin + warp, + WARPS, ... of the range ----
    PagedUnit u = paged_unit_of(start, a.n, a.kv.hkv, g_begin);
    PagedUnit pu = u;
    long long pg = g_begin + warp;                           // next block to copy
    uint32_t issued = 0, consumed = 0, valid = 0;            // valid: bit per stage, the block was copied
    int next_page = -1;
    auto find_page = [&]() {                                 // page id of block pg (loaded ahead of its use)
        if (pg >= g_end) return;
        while (pg >= pu.off + pu.nblk) paged_next_unit(start, a.n, a.kv.hkv, pu);
        next_page = __ldg(a.table + (size_t)pu.b * a.cols + ((int)(pg - pu.off) * BLK >> a.kv.shift));
    };
    auto produce = [&]() {
        if (pg >= g_end) return;
        const int stage = issued % STAGES;
        const int t0 = (int)(pg - pu.off) * BLK;
        const uint32_t bytes = min(BLK, row_length(a, pu.b) - t0) * (D * 2);
        const bool ok = a.kv.has(next_page);
        valid = ok ? valid | 1u << stage : valid & ~(1u << stage);
        if (lane == 0) {
            if (ok) {
                const int layer = a.layer0 + pu.l;
                mbar_arrive_expect_tx(&my_full[stage], 2 * bytes);
                bulk_copy(my_ring + stage * STAGE, a.kv.row(next_page, layer, 0, pu.kh, t0 & mask), bytes, &my_full[stage]);
                bulk_copy(my_ring + stage * STAGE + HALF_STAGE, a.kv.row(next_page, layer, 1, pu.kh, t0 & mask), bytes,
                          &my_full[stage]);
            } else {
                mbar_arrive(&my_full[stage]);
                atomicCAS(a.error, 0, PAGED_BAD_PAGE);
            }
        }
        ++issued;
        pg += WARPS;
        find_page();
    };
    find_page();
    for (int i = 0; i < STAGES; ++i) produce();

    auto load_q = [&](const PagedUnit& w, float4 (&x)[2 * GROUP]) {
        const size_t row = ((size_t)w.l * a.n + w.b) * hq + (size_t)w.kh * GROUP;
        #pragma unroll
        for (int i = 0; i < 2 * GROUP; ++i)
            x[i] = __ldg(reinterpret_cast<const float4*>(a.q + (row + (i >> 1)) * D + sl * 8) + (i & 1));
    };
    float4 q_raw[2 * GROUP];
    load_q(u, q_raw);
    long long my_g = g_begin + warp;                         // next block of this warp to consume
    int parity = 0;
    for (long long g = g_begin; g < g_end; parity ^= 1) {
        const int cnt = (int)(min(u.off + u.nblk, g_end) - g);
        const int len = row_length(a, u.b);
        float2 q[GROUP][4], acc[GROUP][4];
        #pragma unroll
        for (int i = 0; i < GROUP; ++i) {
            const float4 x = q_raw[2 * i], y = q_raw[2 * i + 1];
            q[i][0] = make_float2(x.x * qscale, x.y * qscale); q[i][1] = make_float2(x.z * qscale, x.w * qscale);
            q[i][2] = make_float2(y.x * qscale, y.y * qscale); q[i][3] = make_float2(y.z * qscale, y.w * qscale);
            #pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = make_float2(0.f, 0.f);
        }
        PagedUnit nu = u;                                    // the next segment's queries, loaded meanwhile
        if (g + cnt < g_end) {
            paged_next_unit(start, a.n, a.kv.hkv, nu);
            load_q(nu, q_raw);
        }
        float m = -INFINITY, l = 0.f;                        // of head sl & 1, this lane's share of the sum
        for (; my_g < g + cnt; my_g += WARPS) {
            const int stage = consumed % STAGES;
            bool got = mbar_wait(&my_full[stage], (consumed / STAGES) & 1, &abort_flag);
            if (!got) { abort_flag = 1; atomicCAS(a.error, 0, WAIT_CODE); }
            got = __all_sync(0xffffffffu, got);
            const uint8_t* buf = my_ring + stage * STAGE;
            const int rows = min(BLK, len - (int)(my_g - u.off) * BLK);
            if (got && (valid >> stage & 1)) {
                // row 2i + hw of the block and head gq: partial sums over this lane's 8 channels, then
                // over the 16 lanes; the lane with sl == 2i + gq keeps the logit
                float v[16];
                #pragma unroll
                for (int i = 0; i < BLK / 2; ++i) {
                    float kf[8];
                    unpack8(*reinterpret_cast<const uint4*>(buf + (2 * i + hw) * (D * 2) + sl * 16), kf);
                    #pragma unroll
                    for (int gq = 0; gq < GROUP; ++gq) {
                        float2 d = make_float2(0.f, 0.f);
                        #pragma unroll
                        for (int e = 0; e < 4; ++e) d = ffma2(q[gq][e], make_float2(kf[2 * e], kf[2 * e + 1]), d);
                        v[2 * i + gq] = d.x + d.y;
                    }
                }
                const int t = 2 * (sl >> 1) + hw;            // this lane's row of the block
                const bool there = t < rows;
                float s = transpose_sum16(v, sl);
                if (!there) s = -INFINITY;                   // (stale bytes of the ring)
                if (a.add_weights) a.logits[my_g * (BLK * 2) + t * 2 + (sl & 1)] = s;
                float mb = s;
                #pragma unroll
                for (int o = 2; o <= 16; o <<= 1) mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, o));
                if (__any_sync(0xffffffffu, mb > m)) {
                    const float mn = fmaxf(m, mb);
                    const float scale = exp2_from(m, mn);
                    m = mn;
                    l *= scale;
                    const float other = __shfl_xor_sync(0xffffffffu, scale, 1);
                    const float sc0 = sl & 1 ? other : scale, sc1 = sl & 1 ? scale : other;
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[0][e].x *= sc0; acc[0][e].y *= sc0;
                        acc[1][e].x *= sc1; acc[1][e].y *= sc1;
                    }
                }
                const float p = there ? exp2_from(s, m) : 0.f;
                l += p;
                #pragma unroll
                for (int i = 0; i < BLK / 2; ++i) {
                    uint4 vr = *reinterpret_cast<const uint4*>(buf + HALF_STAGE + (2 * i + hw) * (D * 2) + sl * 16);
                    if (2 * i + hw >= rows) vr = make_uint4(0, 0, 0, 0);   // stale bytes count nothing, whatever they are
                    float vf[8];
                    unpack8(vr, vf);
                    const float p0 = __shfl_sync(0xffffffffu, p, (lane & 16) + 2 * i);
                    const float p1 = __shfl_sync(0xffffffffu, p, (lane & 16) + 2 * i + 1);
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 v2 = make_float2(vf[2 * e], vf[2 * e + 1]);
                        acc[0][e] = ffma2(make_float2(p0, p0), v2, acc[0][e]);
                        acc[1][e] = ffma2(make_float2(p1, p1), v2, acc[1][e]);
                    }
                }
            }
            __syncwarp();                                    // the stage is read by all lanes
            if (got) {
                ++consumed;
                produce();
            }
        }
        // ---- merge the warps ----
        #pragma unroll
        for (int o = 2; o <= 16; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        #pragma unroll
        for (int i = 0; i < GROUP; ++i)
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[i][e].x += __shfl_xor_sync(0xffffffffu, acc[i][e].x, 16);
                acc[i][e].y += __shfl_xor_sync(0xffffffffu, acc[i][e].y, 16);
                if (hw == 0) *reinterpret_cast<float2*>(&s_acc[parity][warp][i][sl * 8 + 2 * e]) = acc[i][e];
            }
        if (lane < 2) { s_stat[parity][warp][lane] = m; s_stat[parity][warp][2 + lane] = l; }
        __syncthreads();                                     // (the other parity's buffers were read before it)
        float M[GROUP], L[GROUP], o[GROUP];
        #pragma unroll
        for (int i = 0; i < GROUP; ++i) {
            M[i] = s_stat[parity][0][i];
            #pragma unroll
            for (int w = 1; w < WARPS; ++w) M[i] = fmaxf(M[i], s_stat[parity][w][i]);
            L[i] = 0.f; o[i] = 0.f;
            #pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = exp2_from(s_stat[parity][w][i], M[i]);
                L[i] += f * s_stat[parity][w][2 + i];
                o[i] += f * s_acc[parity][w][i][tid];
            }
        }
        if (cnt == u.nblk) {
            const size_t qrow = ((size_t)u.l * a.n + u.b) * hq + (size_t)u.kh * GROUP;
            #pragma unroll
            for (int i = 0; i < GROUP; ++i) a.out[(qrow + i) * D + tid] = o[i] / L[i];
            if (a.add_weights) add_weights(a, u, g, cnt, M, L);
        } else {
            float* rec = a.records + ((size_t)c * 2 + (g != g_begin)) * PARTIAL_FLOATS;
            if (tid < GROUP) { rec[tid] = M[tid]; rec[GROUP + tid] = L[tid]; }
            #pragma unroll
            for (int i = 0; i < GROUP; ++i) rec[4 + i * D + tid] = o[i];
        }
        g += cnt;
        u = nu;
    }
    // drain: copies issued but not consumed (after an expired wait) must land before the CTA exits
    for (; consumed < issued; ++consumed) mbar_wait(&my_full[consumed % STAGES], (consumed / STAGES) & 1, &never_abort, 500000000ull);
}

// CTA c joins the unit whose first range is c, and adds the weights of the parts of shared units
// that lie in range c.
__global__ void __launch_bounds__(THREADS) attn_paged_join_kernel(const PagedAttnArgs a) {
    __shared__ int start[MAX_PAGED_BATCH + 1];
    __shared__ int warp_sum[WARPS];
    __shared__ float s_f[CTAS][GROUP];                       // factor of each record
    __shared__ float red[2 * GROUP][WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x, hq = GROUP * a.kv.hkv;
    const PagedSplit sp = scan_lengths(a, start, warp_sum);
    asm volatile("griddepcontrol.wait;" ::: "memory");       // the split launch is complete and its stores visible
    if (sp.total == 0 || c >= sp.ctas) return;
    const long long g_begin = sp.begin(c), g_end = sp.begin(c + 1);
    long long done = -1;
    for (int side = 0; side < 2; ++side) {
        const PagedUnit u = paged_unit_of(start, a.n, a.kv.hkv, side ? g_end - 1 : g_begin);
        if (u.off == done) continue;
        done = u.off;
        const int c_first = sp.range_of(u.off), c_last = sp.range_of(u.off + u.nblk - 1), nrec = c_last - c_first + 1;
        if (nrec == 1 || (c != c_first && !a.add_weights)) continue;
        // record i of the unit: range c_first + i; slot 0 but in the first range, unless it begins the range
        const float* first = a.records + ((size_t)c_first * 2 + (u.off != sp.begin(c_first))) * PARTIAL_FLOATS;
        const float* others = a.records + (size_t)c_first * 2 * PARTIAL_FLOATS;
        float M[GROUP] = {-INFINITY, -INFINITY}, L[GROUP] = {0.f, 0.f};
        __syncthreads();                                     // s_f and red are free
        for (int i = tid; i < nrec; i += THREADS) {
            const float4 st = *reinterpret_cast<const float4*>(i ? others + (size_t)i * 2 * PARTIAL_FLOATS : first);
            M[0] = fmaxf(M[0], st.x); M[1] = fmaxf(M[1], st.y);
        }
        #pragma unroll
        for (int k = 0; k < GROUP; ++k) {
            #pragma unroll
            for (int x = 16; x >= 1; x >>= 1) M[k] = fmaxf(M[k], __shfl_xor_sync(0xffffffffu, M[k], x));
            if (lane == 0) red[k][warp] = M[k];
        }
        __syncthreads();
        #pragma unroll
        for (int k = 0; k < GROUP; ++k)
            #pragma unroll
            for (int w = 0; w < WARPS; ++w) M[k] = fmaxf(M[k], red[k][w]);
        for (int i = tid; i < nrec; i += THREADS) {
            const float4 st = *reinterpret_cast<const float4*>(i ? others + (size_t)i * 2 * PARTIAL_FLOATS : first);
            const float f0 = exp2_from(st.x, M[0]), f1 = exp2_from(st.y, M[1]);
            s_f[i][0] = f0; s_f[i][1] = f1;
            L[0] += f0 * st.z; L[1] += f1 * st.w;
        }
        #pragma unroll
        for (int k = 0; k < GROUP; ++k) {
            #pragma unroll
            for (int x = 16; x >= 1; x >>= 1) L[k] += __shfl_xor_sync(0xffffffffu, L[k], x);
            if (lane == 0) red[GROUP + k][warp] = L[k];
        }
        __syncthreads();
        #pragma unroll
        for (int k = 0; k < GROUP; ++k) {
            L[k] = 0.f;
            #pragma unroll
            for (int w = 0; w < WARPS; ++w) L[k] += red[GROUP + k][w];
        }
        if (c == c_first) {
            float o[GROUP];
            #pragma unroll
            for (int k = 0; k < GROUP; ++k) o[k] = s_f[0][k] * first[4 + k * D + tid];
            #pragma unroll 8
            for (int i = 1; i < nrec; ++i) {
                const float* rec = others + (size_t)i * 2 * PARTIAL_FLOATS + 4 + tid;
                #pragma unroll
                for (int k = 0; k < GROUP; ++k) o[k] += s_f[i][k] * rec[k * D];
            }
            const size_t qrow = ((size_t)u.l * a.n + u.b) * hq + (size_t)u.kh * GROUP;
            #pragma unroll
            for (int k = 0; k < GROUP; ++k) a.out[(qrow + k) * D + tid] = o[k] / L[k];
        }
        if (a.add_weights) {
            const long long g = max(u.off, g_begin);
            add_weights(a, u, g, (int)(min(u.off + u.nblk, g_end) - g), M, L);
        }
    }
}

}  // namespace

size_t paged_attn_record_bytes() { return (size_t)CTAS * 2 * PARTIAL_FLOATS * sizeof(float); }

size_t paged_attn_workspace(int n, int n_layers, int hkv, int max_rows, bool weights) {
    const size_t blocks = (size_t)n * n_layers * hkv * ((max_rows + BLK - 1) / BLK);
    return paged_attn_record_bytes() + (weights ? blocks * BLK * 2 * sizeof(float) : 0);
}

cudaError_t launch_paged_attn(const PagedAttnArgs& a, cudaStream_t s) {
    cudaError_t e = cudaFuncSetAttribute(attn_paged_split_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RING);
    if (e != cudaSuccess) return e;
    attn_paged_split_kernel<<<CTAS, THREADS, RING, s>>>(a);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(CTAS); cfg.blockDim = dim3(THREADS); cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_paged_join_kernel, a);
}

}  // namespace qattn
