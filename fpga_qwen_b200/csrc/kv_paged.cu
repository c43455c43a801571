// kv_paged.cu — fused QK-RMSNorm + RoPE + FP16 write of new rows into the pages of a paged KV cache.
//
// The arithmetic of kv_append.cu, bit for bit (norm_rope.cuh: tampajohn/fpga-qwen
// engine/core.cpp:207-218, :395-405), with each row's place read from device arrays: cache row
// row_len[r] - 1 of table row row_seq[r], RoPE position row_pos[r]. A row whose length is zero is
// padding: nothing is stored and its query rows are zero. Places outside their tables are
// recorded in the error block and skipped.
//
// Layout as in kv_append.cu: a block owns TPB tokens of one layer, one thread per head row (one
// warp); rows are staged in shared memory with 16-byte cp.async copies, the sequential FP64 sum of
// squares runs one row per thread, and the stores are coalesced. Two chains of dependent loads hang
// on the row arrays, position -> RoPE rows and length -> table -> page id; both stay off the
// critical path: the RoPE rows are a second copy group, needed only once the sums are done, and
// the page ids stay in registers that the stores are the first to read.
// HBM-bound: 28,672 algorithmic bytes per (token, layer) at 8 KV heads.
#include "norm_rope.cuh"

namespace qattn {
namespace {

constexpr int STRIDE = 132;       // padded row stride in floats: conflict-free float4 access
constexpr int SLOT = 384;         // staged floats per token: cos[64] sin[64] q_norm[128] k_norm[128]

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)),
                 "l"(gmem) : "memory");
}

template <int HKV, int TPB>
__global__ void __launch_bounds__(TPB * 4 * HKV) kv_paged_append_kernel(const PagedAppendArgs a) {
    constexpr int HQ = GROUP * HKV, R = HQ + 2 * HKV, ROWS = TPB * R;
    static_assert(ROWS == 32, "one warp: the page ids travel by shuffle");
    extern __shared__ __align__(16) float smem[];
    float* tile = smem;                                   // [ROWS][STRIDE]
    float* slots = smem + ROWS * STRIDE;                  // [TPB][SLOT]
    const int l = blockIdx.y, layer = a.layer0 + l;
    const int b0 = blockIdx.x * TPB;
    const int ntok = min(TPB, a.n - b0);
    const int lane = threadIdx.x;
    const size_t tok_base = (size_t)l * a.n + b0;
    const int r_first = a.q_out ? 0 : HQ;                 // without q_out the query rows are not touched

    // lane tb < ntok: the place of token b0 + tb
    int pos = 0, len = 0, seq = 0;
    if (lane < ntok) {
        pos = __ldg(a.row_pos + b0 + lane);
        len = __ldg(a.row_len + b0 + lane);
        seq = a.row_seq ? __ldg(a.row_seq + b0 + lane) : b0 + lane;
    }
    #pragma unroll 8
    for (int row = 0; row < ROWS; ++row) {
        const int tb = row / R, r = row - tb * R;
        if (r < r_first || tb >= ntok) continue;
        const size_t tok = tok_base + tb;
        const float* src = r < HQ ? a.q_pre + (tok * HQ + r) * D
                         : r < HQ + HKV ? a.k_pre + (tok * HKV + (r - HQ)) * D
                                        : a.v_pre + (tok * HKV + (r - HQ - HKV)) * D;
        cp_async16(&tile[row * STRIDE + lane * 4], src + lane * 4);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    #pragma unroll
    for (int tb = 0; tb < TPB; ++tb) {                    // 96 chunks of 16 bytes per token
        if (tb >= ntok) break;
        int p = __shfl_sync(0xffffffffu, pos, tb);
        if ((unsigned)p >= (unsigned)a.rope_rows) p = 0;  // recorded and skipped below
        cp_async16(&slots[tb * SLOT + lane * 4], lane < 16 ? a.cosines + (size_t)p * 64 + lane * 4
                                                           : a.sines + (size_t)p * 64 + (lane - 16) * 4);
        #pragma unroll
        for (int c = 0; c < 2; ++c)
            cp_async16(&slots[tb * SLOT + 128 + c * D + lane * 4], a.norms + ((size_t)layer * 2 + c) * D + lane * 4);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    int code = 0, page = -1;
    if (lane < ntok)
        page = paged_place(len, seq, pos, a.n_seqs, a.cols, a.kv.shift, a.rope_rows, a.kv.n_pages, a.table, &code);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();

    {
        const int tb = lane / R, r = lane - tb * R;
        const bool turn = tb < ntok && r >= r_first && r < HQ + HKV;
        float* x = &tile[lane * STRIDE];
        const float inv = turn ? rms_inv(x, a.eps) : 0.f;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        if (turn) {
            const float* slot = &slots[tb * SLOT];
            norm_rope_row(x, slot + 128 + (r < HQ ? 0 : D), slot, slot + 64, inv);
        }
    }
    __syncwarp();

    if (code) atomicCAS(a.error, 0, code);
    const int at = (int)(((unsigned)len - 1u) & ((1u << a.kv.shift) - 1u));
    #pragma unroll 4
    for (int row = 0; row < ROWS; ++row) {
        const int tb = row / R, r = row - tb * R;
        if (r < r_first || tb >= ntok) continue;
        const float* x = &tile[row * STRIDE];
        const int pg = __shfl_sync(0xffffffffu, page, tb), t = __shfl_sync(0xffffffffu, at, tb);
        if (r < HQ) {
            float* dst = a.q_out + ((tok_base + tb) * HQ + r) * D;
            reinterpret_cast<float4*>(dst)[lane] =
                pg < 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(x + lane * 4);
        } else if (pg >= 0) {
            const int kind = r < HQ + HKV ? 0 : 1;
            const int head = r - HQ - kind * HKV;
            if (lane < 16)
                reinterpret_cast<uint4*>(a.kv.row(pg, layer, kind, head, t))[lane] = half8_rn(x + lane * 8);
            else if (lane == 16 && kind == 0 && a.kv.weights)
                *a.kv.weight(pg, layer, head, t) = 0.f;
        }
    }
}

template <int HKV, int TPB>
void launch_t(const PagedAppendArgs& a, cudaStream_t s) {
    constexpr int ROWS = TPB * 4 * HKV;
    constexpr size_t smem = ((size_t)ROWS * STRIDE + (size_t)TPB * SLOT) * sizeof(float);
    static_assert(smem <= 48 << 10, "within the default shared-memory limit");
    const dim3 grid((a.n + TPB - 1) / TPB, a.n_layers);
    kv_paged_append_kernel<HKV, TPB><<<grid, ROWS, smem, s>>>(a);
}

}  // namespace

void launch_paged_append(const PagedAppendArgs& a, cudaStream_t s) {
    switch (a.kv.hkv) {
        case 8: launch_t<8, 1>(a, s); break;
        case 4: launch_t<4, 2>(a, s); break;
        case 2: launch_t<2, 4>(a, s); break;
        case 1: launch_t<1, 8>(a, s); break;
        default: break;   // rejected at context creation
    }
}

}  // namespace qattn
