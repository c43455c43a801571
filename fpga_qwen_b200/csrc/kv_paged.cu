// kv_paged.cu — fused QK-RMSNorm + RoPE + FP16 write of new rows into the pages of a paged KV cache.
//
// The arithmetic of kv_append.cu, bit for bit (norm_rope.cuh: tampajohn/fpga-qwen
// engine/core.cpp:207-218, :395-405), with each row's place read from device arrays: cache row
// row_len[r] - 1 of table row row_seq[r], RoPE position row_pos[r]. A row whose length is zero is
// padding: nothing is stored and its query rows are zero. Places outside their tables are
// recorded in the error block and skipped.
//
// One warp takes TPB tokens of one layer, 32 head rows. Query and key rows are staged in shared
// memory with 16-byte cp.async copies for the sequential FP64 sum of squares, one row per lane;
// then the warp goes through them row by row, a lane normalising and rotating channels 2l, 2l + 1
// and their partners 64 above, whose RoPE values and norm weights it holds in registers, and
// storing them. Value rows pass through registers only. HBM-bound (28,672 algorithmic bytes per
// (token, layer) at 8 KV heads), if there are few enough instructions and enough warps: staging
// everything and rotating one row per thread, as kv_append.cu does, took twice the instructions and
// a third more shared memory, and 612 us for 3968 tokens x 28 layers.
// Two chains of dependent loads hang on the row arrays, position -> RoPE values and length ->
// table -> page id; both are in flight beside the rows.
// Launches overlap (programmatic dependent launch): a small append, of a step, lets the attention behind it
// start at once and itself starts behind the attention before it (28 layers layer by layer: 1 row of 448,
// 324 -> 309 us; 8 rows of 300, 356 -> 340 us). Large ones let the next launch start as they end: its
// waiting warps would take the place of theirs (64 rows x 28 layers 10.4 -> 11.8 us).
#include "norm_rope.cuh"

namespace qattn {
namespace {

constexpr int STRIDE = 132;       // padded row stride in floats: conflict-free float4 access

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)),
                 "l"(gmem) : "memory");
}

__device__ __forceinline__ float2 load2(const float* p) { return *reinterpret_cast<const float2*>(p); }

template <int HKV, int TPB>
__global__ void __launch_bounds__(32) kv_paged_append_kernel(const PagedAppendArgs a) {
    constexpr int HQ = GROUP * HKV, QK = HQ + HKV, ROWS = TPB * QK;   // staged rows: [token][query heads | key heads]
    static_assert(TPB * (QK + HKV) == 32 && ROWS == 24, "one warp: 24 query and key rows, 8 value rows");
    __shared__ __align__(16) float tile[ROWS][STRIDE];
    const int l = blockIdx.y, layer = a.layer0 + l;
    const int b0 = blockIdx.x * TPB;
    const int ntok = min(TPB, a.n - b0);
    const int lane = threadIdx.x;
    const size_t tok_base = (size_t)l * a.n + b0;
    const bool with_q = a.q_out != nullptr;               // without q_out the query rows are not touched

    // What ran before is complete. (No read-only loads below: they may move across this.)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (gridDim.x * gridDim.y <= 2 * NUM_SMS_B200) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // lane tb < ntok: the place of token b0 + tb
    int pos = 0, len = 0, seq = 0;
    if (lane < ntok) {
        pos = a.row_pos[b0 + lane];
        len = a.row_len[b0 + lane];
        seq = a.row_seq ? a.row_seq[b0 + lane] : b0 + lane;
    }
    #pragma unroll
    for (int row = 0; row < ROWS; ++row) {
        const int tb = row / QK, r = row - tb * QK;
        if (tb >= ntok || (r < HQ && !with_q)) continue;
        const float* src = r < HQ ? a.q_pre + ((tok_base + tb) * HQ + r) * D : a.k_pre + ((tok_base + tb) * HKV + (r - HQ)) * D;
        cp_async16(&tile[row][lane * 4], src + lane * 4);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    // value rows: two at a time, 8 channels a lane; row 2i + lane / 16 of the tokens' TPB * HKV
    float4 v[4][2];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 2 * i + (lane >> 4);
        if (row / HKV < ntok) {
            const float4* src = reinterpret_cast<const float4*>(a.v_pre + (tok_base * HKV + row) * D) + (lane & 15) * 2;
            v[i][0] = src[0];
            v[i][1] = src[1];
        }
    }
    const float* norms = a.norms + (size_t)layer * 2 * D + 2 * lane;
    const float2 wq0 = load2(norms), wq1 = load2(norms + 64), wk0 = load2(norms + D), wk1 = load2(norms + D + 64);
    float2 cs[TPB], sn[TPB];
    #pragma unroll
    for (int tb = 0; tb < TPB; ++tb) {
        int p = __shfl_sync(0xffffffffu, pos, tb);
        if ((unsigned)p >= (unsigned)a.rope_rows) p = 0;  // recorded and skipped below
        cs[tb] = load2(a.cosines + (size_t)p * 64 + 2 * lane);
        sn[tb] = load2(a.sines + (size_t)p * 64 + 2 * lane);
    }
    int code = 0, page = -1;
    if (lane < ntok)
        page = paged_place(len, seq, pos, a.n_seqs, a.cols, a.kv.shift, a.rope_rows, a.kv.n_pages, a.table, &code);
    if (code) atomicCAS(a.error + ERR_DATA, 0, code);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    float inv = 0.f;                                      // of row `lane`
    if (lane < ROWS && lane / QK < ntok && (with_q || lane % QK >= HQ)) inv = rms_inv(tile[lane], a.eps);

    const int at = (int)(((unsigned)len - 1u) & ((1u << a.kv.shift) - 1u));
    #pragma unroll
    for (int tb = 0; tb < TPB; ++tb) {
        if (tb >= ntok) break;
        const int pg = __shfl_sync(0xffffffffu, page, tb), t = __shfl_sync(0xffffffffu, at, tb);
        // the token's first key row; heads are 1 << shift rows apart, values hkv heads behind keys
        __half* const k_row = a.kv.row(max(pg, 0), layer, 0, 0, t);
        const size_t head_step = (size_t)D << a.kv.shift;
        if (with_q) {
            float* const q_row = a.q_out + (tok_base + tb) * HQ * D + 2 * lane;
            #pragma unroll 8
            for (int h = 0; h < HQ; ++h) {
                const float* x = tile[tb * QK + h] + 2 * lane;
                const float2 x0 = *reinterpret_cast<const float2*>(x), x1 = *reinterpret_cast<const float2*>(x + 64);
                const float f = __shfl_sync(0xffffffffu, inv, tb * QK + h);
                float2 r0, r1;
                norm_rope_pair(x0.x, x1.x, wq0.x, wq1.x, cs[tb].x, sn[tb].x, f, r0.x, r1.x);
                norm_rope_pair(x0.y, x1.y, wq0.y, wq1.y, cs[tb].y, sn[tb].y, f, r0.y, r1.y);
                if (pg < 0) r0 = r1 = make_float2(0.f, 0.f);
                *reinterpret_cast<float2*>(q_row + h * D) = r0;
                *reinterpret_cast<float2*>(q_row + h * D + 64) = r1;
            }
        }
        #pragma unroll
        for (int h = 0; h < HKV; ++h) {
            const float* x = tile[tb * QK + HQ + h] + 2 * lane;
            const float2 x0 = *reinterpret_cast<const float2*>(x), x1 = *reinterpret_cast<const float2*>(x + 64);
            const float f = __shfl_sync(0xffffffffu, inv, tb * QK + HQ + h);
            float2 r0, r1;
            norm_rope_pair(x0.x, x1.x, wk0.x, wk1.x, cs[tb].x, sn[tb].x, f, r0.x, r1.x);
            norm_rope_pair(x0.y, x1.y, wk0.y, wk1.y, cs[tb].y, sn[tb].y, f, r0.y, r1.y);
            if (pg >= 0) {
                __half2* const to = reinterpret_cast<__half2*>(k_row + h * head_step) + lane;
                to[0] = __floats2half2_rn(r0.x, r0.y);
                to[32] = __floats2half2_rn(r1.x, r1.y);
            }
        }
        if (pg >= 0 && a.kv.weights && lane < HKV) *a.kv.weight(pg, layer, lane, t) = 0.f;
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 2 * i + (lane >> 4), tb = row / HKV;
        const int pg = __shfl_sync(0xffffffffu, page, tb), t = __shfl_sync(0xffffffffu, at, tb);
        if (tb < ntok && pg >= 0)
            reinterpret_cast<uint4*>(a.kv.row(pg, layer, 1, row - tb * HKV, t))[lane & 15] =
                half8_rn(v[i][0], v[i][1]);
    }
}

template <int HKV>
void launch_t(const PagedAppendArgs& a, cudaStream_t s) {
    constexpr int TPB = 8 / HKV;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((a.n + TPB - 1) / TPB, a.n_layers); cfg.blockDim = dim3(32); cfg.stream = s;
    cfg.attrs = &attr; cfg.numAttrs = a.overlap ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kv_paged_append_kernel<HKV, TPB>, a);   // (errors: after_launch)
}

}  // namespace

void launch_paged_append(const PagedAppendArgs& a, cudaStream_t s) {
    switch (a.kv.hkv) {
        case 8: launch_t<8>(a, s); break;
        case 4: launch_t<4>(a, s); break;
        case 2: launch_t<2>(a, s); break;
        case 1: launch_t<1>(a, s); break;
        default: break;   // rejected at context creation
    }
}

}  // namespace qattn
