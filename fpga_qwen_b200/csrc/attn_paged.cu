// attn_paged.cu — decode attention of one query row per sequence over a paged KV cache.
//
// For row b with L = lengths[b] cached rows, layer l and KV head kh, both query heads h of the
// group: s_t = q_h . k_t / sqrt(128), p = softmax(s), out_h = sum_t p_t v_t, all in FP32 over the
// FP16 rows; with add_weights also weights[t] += p_t of both heads.
//
// Even split (stream-K style): the 16-row blocks of all (layer, row, KV head) units are laid end
// to end and cut into equal ranges, one per CTA, whatever the lengths are; lengths are read on
// the device, so every CTA first scans them. A range can end inside one unit and continue in the
// next. Each warp takes every fourth block of the CTA's part of a unit (a segment) with its own
// running maximum and sum; the CTA merges its warps at the segment's end. A unit inside one range
// is finished there; a unit that several ranges share leaves one record (max, sum, 2 x 128
// partial output) per range, and a second launch joins them in range order (no atomics, so the
// result does not depend on timing). At most two units of a range are shared (its first and its
// last), so the records are 2 per CTA, whatever the batch.
//
// The weights need the final maximum and sum: the logits go to the workspace (8 bytes a row and
// KV head against 512 of K and V) and become weights when the unit is finished, in this launch or
// in the joining one. Each (row, KV head) weight gets one FP32 addition.
#include "qattn_common.cuh"
#include "sm100.cuh"

namespace qattn {
namespace {

constexpr int THREADS = 128, WARPS = THREADS / 32;
constexpr int BLK = PAGED_BLK;
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

__global__ void __launch_bounds__(THREADS, 2) attn_paged_split_kernel(const PagedAttnArgs a) {
    __shared__ int start[MAX_PAGED_BATCH + 1];
    __shared__ int warp_sum[WARPS];
    __shared__ float s_stat[WARPS][4];                       // per warp: max and sum of both heads
    __shared__ __align__(16) float s_acc[WARPS][GROUP][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hw = lane >> 4, sl = lane & 15;                // half-warp: rows of one parity; 8 channels a lane
    const int hq = GROUP * a.kv.hkv;
    const PagedSplit sp = scan_lengths(a, start, warp_sum);
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

    PagedUnit u = paged_unit_of(start, a.n, a.kv.hkv, g_begin);
    for (long long g = g_begin; g < g_end;) {
        if (g != g_begin) paged_next_unit(start, a.n, a.kv.hkv, u);
        const int blk0 = (int)(g - u.off);
        const int cnt = (int)(min(u.off + u.nblk, g_end) - g);
        const int len = row_length(a, u.b), layer = a.layer0 + u.l;
        const size_t qrow = ((size_t)u.l * a.n + u.b) * hq + (size_t)u.kh * GROUP;
        float q[GROUP][8], acc[GROUP][8];
        #pragma unroll
        for (int i = 0; i < GROUP; ++i) {
            const float4* src = reinterpret_cast<const float4*>(a.q + (qrow + i) * D + sl * 8);
            const float4 x = __ldg(src), y = __ldg(src + 1);
            q[i][0] = x.x * qscale; q[i][1] = x.y * qscale; q[i][2] = x.z * qscale; q[i][3] = x.w * qscale;
            q[i][4] = y.x * qscale; q[i][5] = y.y * qscale; q[i][6] = y.z * qscale; q[i][7] = y.w * qscale;
            #pragma unroll
            for (int e = 0; e < 8; ++e) acc[i][e] = 0.f;
        }
        float m = -INFINITY, l = 0.f;                        // of head sl & 1, this lane's share of the sum
        for (int j = warp; j < cnt; j += WARPS) {
            const int t0 = (blk0 + j) * BLK, rows = min(BLK, len - t0);
            const int page = a.table[(size_t)u.b * a.cols + (t0 >> a.kv.shift)];
            if (!a.kv.has(page)) {
                if (lane == 0) atomicCAS(a.error, 0, PAGED_BAD_PAGE);
                continue;
            }
            const uint4* K = reinterpret_cast<const uint4*>(a.kv.row(page, layer, 0, u.kh, t0 & mask));
            const uint4* V = reinterpret_cast<const uint4*>(a.kv.row(page, layer, 1, u.kh, t0 & mask));
            // row 2i + hw of the block, head gq: this lane's 8 channels, then the sum over 16 lanes
            float s = -INFINITY;                             // kept by the lane with sl == 2i + gq
            #pragma unroll
            for (int i = 0; i < BLK / 2; ++i) {
                const int t = 2 * i + hw;
                uint4 kr = make_uint4(0, 0, 0, 0);
                if (t < rows) kr = K[t * 16 + sl];
                float kf[8];
                unpack8(kr, kf);
                #pragma unroll
                for (int gq = 0; gq < GROUP; ++gq) {
                    float d = 0.f;
                    #pragma unroll
                    for (int e = 0; e < 8; ++e) d = fmaf(q[gq][e], kf[e], d);
                    #pragma unroll
                    for (int o = 8; o >= 1; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                    if (sl == 2 * i + gq && t < rows) s = d;
                }
            }
            if (a.add_weights) a.logits[(g + j) * (BLK * 2) + (2 * (sl >> 1) + hw) * 2 + (sl & 1)] = s;
            float mb = s;
            #pragma unroll
            for (int o = 2; o <= 16; o <<= 1) mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, o));
            const float mn = fmaxf(m, mb);
            const float scale = exp2_from(m, mn);
            const bool there = 2 * (sl >> 1) + hw < rows;
            const float p = there ? exp2_from(s, mn) : 0.f;
            m = mn;
            l = l * scale + p;
            const float other = __shfl_xor_sync(0xffffffffu, scale, 1);
            const float sc0 = sl & 1 ? other : scale, sc1 = sl & 1 ? scale : other;
            #pragma unroll
            for (int e = 0; e < 8; ++e) { acc[0][e] *= sc0; acc[1][e] *= sc1; }
            #pragma unroll
            for (int i = 0; i < BLK / 2; ++i) {
                const int t = 2 * i + hw;
                uint4 vr = make_uint4(0, 0, 0, 0);           // rows past the length count nothing, whatever they hold
                if (t < rows) vr = V[t * 16 + sl];
                float vf[8];
                unpack8(vr, vf);
                const float p0 = __shfl_sync(0xffffffffu, p, (lane & 16) + 2 * i);
                const float p1 = __shfl_sync(0xffffffffu, p, (lane & 16) + 2 * i + 1);
                #pragma unroll
                for (int e = 0; e < 8; ++e) { acc[0][e] = fmaf(p0, vf[e], acc[0][e]); acc[1][e] = fmaf(p1, vf[e], acc[1][e]); }
            }
        }
        // ---- merge the warps ----
        #pragma unroll
        for (int o = 2; o <= 16; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        #pragma unroll
        for (int i = 0; i < GROUP; ++i)
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                acc[i][e] += __shfl_xor_sync(0xffffffffu, acc[i][e], 16);
                if (hw == 0) s_acc[warp][i][sl * 8 + e] = acc[i][e];
            }
        if (lane < 2) { s_stat[warp][lane] = m; s_stat[warp][2 + lane] = l; }
        __syncthreads();
        float M[GROUP], L[GROUP], o[GROUP];
        #pragma unroll
        for (int i = 0; i < GROUP; ++i) {
            M[i] = s_stat[0][i];
            for (int w = 1; w < WARPS; ++w) M[i] = fmaxf(M[i], s_stat[w][i]);
            L[i] = 0.f; o[i] = 0.f;
            for (int w = 0; w < WARPS; ++w) {
                const float f = exp2_from(s_stat[w][i], M[i]);
                L[i] += f * s_stat[w][2 + i];
                o[i] += f * s_acc[w][i][tid];
            }
        }
        if (cnt == u.nblk) {
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
        __syncthreads();                                     // s_acc, s_stat and the logits are read
    }
}

// CTA c joins the unit whose first range is c, and adds the weights of the parts of shared units
// that lie in range c.
__global__ void __launch_bounds__(THREADS) attn_paged_join_kernel(const PagedAttnArgs a) {
    __shared__ int start[MAX_PAGED_BATCH + 1];
    __shared__ int warp_sum[WARPS];
    const int tid = threadIdx.x, c = blockIdx.x, hq = GROUP * a.kv.hkv;
    const PagedSplit sp = scan_lengths(a, start, warp_sum);
    if (sp.total == 0 || c >= sp.ctas) return;
    const long long g_begin = sp.begin(c), g_end = sp.begin(c + 1);
    long long done = -1;
    for (int side = 0; side < 2; ++side) {
        const PagedUnit u = paged_unit_of(start, a.n, a.kv.hkv, side ? g_end - 1 : g_begin);
        if (u.off == done) continue;
        done = u.off;
        const int c_first = sp.range_of(u.off), c_last = sp.range_of(u.off + u.nblk - 1);
        if (c_first == c_last || (c != c_first && !a.add_weights)) continue;
        float M[GROUP] = {-INFINITY, -INFINITY}, L[GROUP] = {0.f, 0.f}, o[GROUP] = {0.f, 0.f};
        for (int r = c_first; r <= c_last; ++r) {
            const float* rec = a.records + ((size_t)r * 2 + (r == c_first && u.off != sp.begin(r))) * PARTIAL_FLOATS;
            #pragma unroll
            for (int i = 0; i < GROUP; ++i) {
                const float mn = fmaxf(M[i], rec[i]);
                const float f = exp2_from(M[i], mn), fr = exp2_from(rec[i], mn);
                M[i] = mn;
                L[i] = L[i] * f + rec[GROUP + i] * fr;
                o[i] = o[i] * f + rec[4 + i * D + tid] * fr;
            }
        }
        if (c == c_first) {
            const size_t qrow = ((size_t)u.l * a.n + u.b) * hq + (size_t)u.kh * GROUP;
            #pragma unroll
            for (int i = 0; i < GROUP; ++i) a.out[(qrow + i) * D + tid] = o[i] / L[i];
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
    attn_paged_split_kernel<<<CTAS, THREADS, 0, s>>>(a);
    attn_paged_join_kernel<<<CTAS, THREADS, 0, s>>>(a);
    return cudaSuccess;
}

}  // namespace qattn
