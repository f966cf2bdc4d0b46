// Attention of new tokens over the paged cache (vqa_paged_attn_*).
#include <algorithm>

#include "vqa_paged_attn.h"

namespace vqa {
namespace paged {

// One wave per row and query head.
template <typename Tag, int D, bool kE4m3>
__global__ __launch_bounds__(256) void rows_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = (int)(id / a.Hq), hq = (int)(id % a.Hq);
    if (row >= a.g.T) return;
    const int s = find_seq(a.g, row, lane);
    if (s >= a.g.S) return;
    const Seq q = seq_of(a.g, s);
    if (row < q.q0 || row >= q.q0 + q.n) return;
    const Range r = visible(a, q, row - q.q0);
    RowState<D> st;
    row_by_lanes<Tag, D, kE4m3>(a, s, hq / a.G, a.q + (int64_t)row * a.q_st + (int64_t)hq * a.q_sh, r.lo, r.hi, st, lane);
    store_row<Tag, D>(a, st, row, hq, lane);
}

template <typename Tag, int D, bool kE4m3>
int launch(const AttnArgs& a, hipStream_t stream) {
    const int64_t blocks = ((int64_t)a.g.T * a.Hq + 3) / 4;
    rows_kernel<Tag, D, kE4m3><<<dim3((unsigned)blocks), 256, 0, stream>>>(a);
    return launch_status();
}

template <typename Tag>
int attn(const void* q, const void* k_pages, const void* v_pages, const uint8_t* k_exp, const uint8_t* v_exp,
         const int32_t* table, const int32_t* cu, const int32_t* lens, void* out, float* lse, void* ws, size_t ws_bytes,
         int T, int S, int Hq, int Hkv, int D, int page, int n_pages, int width, int e4m3, const int64_t* st, int causal,
         int window, int max_q, float scale, hipStream_t stream) {
    if (!q || !k_pages || !v_pages || !table || !cu || !lens || !out || !st) return VQA_ERR_NULL_POINTER;
    if (Hkv < 1 || Hq < 1 || Hq % Hkv || Hq > 65535 || (int64_t)T * Hq > (int64_t(1) << 31) - 1) return VQA_ERR_BAD_SHAPE;
    if (D != 64 && D != 128) return VQA_ERR_UNSUPPORTED_HEAD_DIM;
    if (window >= 0 && !causal) return VQA_ERR_BAD_ARGUMENT;
    if (!(scale > 0.f) || !(scale <= 3e38f)) return VQA_ERR_BAD_ARGUMENT;
    AttnArgs a{};
    if (int rc = make_seqs(&a.g, cu, lens, table, st[12], S, T, width, n_pages, page)) return rc;
    if (int rc = make_pool(&a.kp, k_pages, k_exp, st + 2, st + 8, e4m3, page)) return rc;
    if (int rc = make_pool(&a.vp, v_pages, v_exp, st + 5, st + 10, e4m3, page)) return rc;
    if (!aligned16(q) || !aligned16(out) || (st[0] | st[1] | st[13] | st[14]) % 8) return VQA_ERR_MISALIGNED;
    a.q = (const uint16_t*)q, a.q_st = st[0], a.q_sh = st[1];
    a.out = (uint16_t*)out, a.o_st = st[13], a.o_sh = st[14];
    a.lse = lse;
    a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv;
    a.causal = causal != 0;
    a.window = window < 0 ? 1 << 30 : std::min(window, 1 << 30);
    a.scale_log2e = scale * kLog2e;
    if (S == 0 || T == 0) return VQA_OK;
    if (D == 128) return e4m3 ? launch<Tag, 128, true>(a, stream) : launch<Tag, 128, false>(a, stream);
    return e4m3 ? launch<Tag, 64, true>(a, stream) : launch<Tag, 64, false>(a, stream);
}

}  // namespace paged
}  // namespace vqa

extern "C" {

size_t vqa_paged_attn_workspace_bytes(int T, int S, int Hq, int Hkv, int D, int max_q) { return 0; }

#define VQA_PAGED_ATTN(sfx, tag)                                                                                          \
    int vqa_paged_attn_##sfx(const void* q, const void* k_pages, const void* v_pages, const uint8_t* k_exp,              \
                             const uint8_t* v_exp, const int32_t* block_table, const int32_t* cu_q,                       \
                             const int32_t* kv_lens, void* out, float* lse, void* workspace, size_t workspace_bytes,      \
                             int T, int S, int Hq, int Hkv, int D, int page, int n_pages, int width, int e4m3,            \
                             const int64_t* strides, int causal, int window, int max_q, float sm_scale,                   \
                             vqa_stream_t stream) {                                                                       \
        return vqa::paged::attn<vqa::tag>(q, k_pages, v_pages, k_exp, v_exp, block_table, cu_q, kv_lens, out, lse,        \
                                          workspace, workspace_bytes, T, S, Hq, Hkv, D, page, n_pages, width, e4m3,       \
                                          strides, causal, window, max_q, sm_scale, stream);                              \
    }

VQA_PAGED_ATTN(bf16, bf16_tag)
VQA_PAGED_ATTN(f16, f16_tag)

}  // extern "C"
