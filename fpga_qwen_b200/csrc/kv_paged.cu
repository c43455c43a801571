// kv_paged.cu — fused QK-RMSNorm + RoPE + FP16 write of new rows into the pages of a paged KV cache.
//
// The arithmetic of kv_append.cu, bit for bit (norm_rope.cuh: tampajohn/fpga-qwen
// engine/core.cpp:207-218, :395-405), with each row's place read from device arrays: cache row
// row_len[r] - 1 of table row row_seq[r], RoPE position row_pos[r]. A row whose length is zero is
// padding: nothing is stored and its query rows are zero. Places outside their tables are
// recorded in the error block and skipped.
//
// Layout as in kv_append.cu: a block owns TPB tokens of one layer, one thread per head row; rows,
// RoPE rows and norm weights are staged in shared memory with 16-byte cp.async copies, the
// sequential FP64 sum of squares runs one row per thread, and the stores are coalesced. The
// table look-up (row_len -> page id) runs on one thread per token while the copies are in flight.
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
    constexpr int HQ = GROUP * HKV, R = HQ + 2 * HKV, ROWS = TPB * R, WARPS = (ROWS + 31) / 32;
    extern __shared__ __align__(16) float smem[];
    float* tile = smem;                                   // [ROWS][STRIDE]
    float* slots = smem + ROWS * STRIDE;                  // [TPB][SLOT]
    __shared__ int s_page[TPB], s_row[TPB];               // page < 0: nothing to store
    const int l = blockIdx.y, layer = a.layer0 + l;
    const int b0 = blockIdx.x * TPB;
    const int ntok = min(TPB, a.n - b0);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t tok_base = (size_t)l * a.n + b0;
    const int r_first = a.q_out ? 0 : HQ;                 // without q_out the query rows are not touched

    for (int row = warp; row < ntok * R; row += WARPS) {
        const int tb = row / R, r = row - tb * R;
        if (r < r_first) continue;
        const size_t tok = tok_base + tb;
        const float* src = r < HQ ? a.q_pre + (tok * HQ + r) * D
                         : r < HQ + HKV ? a.k_pre + (tok * HKV + (r - HQ)) * D
                                        : a.v_pre + (tok * HKV + (r - HQ - HKV)) * D;
        cp_async16(&tile[row * STRIDE + lane * 4], src + lane * 4);
    }
    for (int i = threadIdx.x; i < ntok * (SLOT / 4); i += ROWS) {
        const int tb = i / (SLOT / 4), c = i - tb * (SLOT / 4);   // 96 chunks of 16 bytes per token
        int pos = a.row_pos[b0 + tb];
        if ((unsigned)pos >= (unsigned)a.rope_rows) pos = 0;      // recorded and skipped below
        const float* src = c < 16 ? a.cosines + (size_t)pos * 64 + c * 4
                         : c < 32 ? a.sines + (size_t)pos * 64 + (c - 16) * 4
                                  : a.norms + (size_t)layer * 2 * D + (c - 32) * 4;
        cp_async16(&slots[tb * SLOT + c * 4], src);
    }
    if (threadIdx.x < ntok) {
        const int b = b0 + threadIdx.x;
        const int len = a.row_len[b], seq = a.row_seq ? a.row_seq[b] : b;
        int code;
        const int page = paged_place(len, seq, a.row_pos[b], a.n_seqs, a.cols, a.kv.shift, a.rope_rows, a.kv.n_pages,
                                     a.table, &code);
        if (code) atomicCAS(a.error, 0, code);
        s_page[threadIdx.x] = page;
        s_row[threadIdx.x] = (int)(((unsigned)len - 1u) & ((1u << a.kv.shift) - 1u));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();

    {
        const int row = threadIdx.x;
        const int tb = row / R, r = row - tb * R;
        if (tb < ntok && r >= r_first && r < HQ + HKV) {
            const float* slot = &slots[tb * SLOT];
            norm_rope_row(&tile[row * STRIDE], slot + 128 + (r < HQ ? 0 : D), slot, slot + 64, a.eps);
        }
    }
    __syncthreads();

    for (int row = warp; row < ntok * R; row += WARPS) {
        const int tb = row / R, r = row - tb * R;
        if (r < r_first) continue;
        const float* x = &tile[row * STRIDE];
        const int page = s_page[tb];
        if (r < HQ) {
            float* dst = a.q_out + ((tok_base + tb) * HQ + r) * D;
            reinterpret_cast<float4*>(dst)[lane] =
                page < 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(x + lane * 4);
        } else if (page >= 0) {
            const int kind = r < HQ + HKV ? 0 : 1;
            const int head = r - HQ - kind * HKV;
            if (lane < 16)
                reinterpret_cast<uint4*>(a.kv.row(page, layer, kind, head, s_row[tb]))[lane] = half8_rn(x + lane * 8);
            else if (lane == 16 && kind == 0 && a.kv.weights)
                *a.kv.weight(page, layer, head, s_row[tb]) = 0.f;
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
