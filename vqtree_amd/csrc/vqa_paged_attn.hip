// Attention of new tokens over the paged cache (vqa_paged_attn_*).
#include <algorithm>

#include "vqa_paged_attn.h"

namespace vqa {
namespace paged {

// Joins the splits of a row: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.  One workgroup per row and query head,
// its waves share the splits (their partial rows are 512 bytes each, so what counts is how many are in flight).
constexpr int kJoinWaves = 4;

template <typename Tag, int D>
__global__ __launch_bounds__(kJoinWaves * 64) void join_kernel(AttnArgs a, Plan few, Plan chunk) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = (int)(blockIdx.x / (unsigned)a.Hq), hq = (int)(blockIdx.x % (unsigned)a.Hq);
    const int s = find_seq(a.g, row, lane);
    if (s >= a.g.S) return;
    const Seq q = seq_of(a.g, s);
    if (row < q.q0 || row >= q.q0 + q.n) return;
    const Plan p = tiles_of(a, few, q) ? few : chunk;
    if (p.parts == 0) return;  // (whole tiles)
    Line line;
    line.init(a, p, lane);
    int tile = 0;  // number of the row's tile: the tiles of the sequences before it, then its own
    for (int base = 0; base < s; base += kWave) {
        const int mine = base + lane < s ? tiles_of(a, p, seq_of(a.g, base + lane)) : 0;
        tile += __builtin_amdgcn_readlane(scan32(mine, lane), 63);
    }
    const int h = hq / a.G, r = (row - q.q0) * a.G + hq % a.G;
    int n_steps;
    const int64_t from = line.start_of_tile(a, p, tile + r / p.rows, n_steps, lane);
    const int i0 = line.part_of(from), i1 = line.part_of(from + n_steps - 1);
    if (i0 == i1) return;  // (one workgroup had the whole tile and has stored the result)
    // the tile is the first piece of every part it reaches but perhaps the one it begins in
    const int shift = from == line.start(i0) ? 0 : 1;
    auto place = [&](int i) { return ((int64_t)(2 * i + (i == i0 ? shift : 0)) * a.Hkv + h) * p.rows + r % p.rows; };
    float top = -INFINITY;
    for (int i = i0 + lane; i <= i1; i += 64) top = fmaxf(top, p.ml[place(i) * 2]);
    top = wave_max(top);
    float o[E], l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
    for (int i = i0 + wave; i <= i1; i += kJoinWaves) {
        const int64_t at = place(i);
        const float m = p.ml[at * 2];
        const float f = m == -INFINITY ? 0.f : fast_exp2(m - top);
        l += f * p.ml[at * 2 + 1];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += f * p.o[at * D + lane * E + e];
    }
    __shared__ float part[kJoinWaves][64][E + 1];
#pragma unroll
    for (int e = 0; e < E; ++e) part[wave][lane][e] = o[e];
    part[wave][lane][E] = l;
    __syncthreads();
    if (wave != 0) return;
    RowState<D> st;
    st.m = top, st.l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) st.o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
        st.l += part[w][lane][E];
#pragma unroll
        for (int e = 0; e < E; ++e) st.o[e] += part[w][lane][e];
    }
    store_row<Tag, D>(a, st, row, hq, lane);
}

// How a call is cut up (host side; how many rows and keys there are is known on the device only).
struct Cut {
    Plan few, chunk;                // (a plan without rows: its kernel is not needed)
    int64_t few_grid, chunk_grid;
    size_t few_bytes, chunk_bytes;  // workspace
};

constexpr int kCus = 256;           // workgroups that fill the chip: one per compute unit, in both kernels
constexpr int kWholeSteps = 32;     // a tile of so few key steps is not worth a split and the launch that joins it
constexpr int kFewRows = 64;        // sequences of more rows go to the chunk kernel

inline size_t round256(size_t x) { return (x + 255) & ~size_t(255); }
inline size_t o_bytes(const Plan& p, int Hkv, int D) { return round256((size_t)2 * p.parts * Hkv * p.rows * D * 4); }
inline size_t ml_bytes(const Plan& p, int Hkv) { return round256((size_t)2 * p.parts * Hkv * p.rows * 8); }

// keys: most keys a row can see, as far as the caller's numbers tell
inline Cut cut_call(int T, int S, int Hq, int Hkv, int D, int max_q, int64_t keys, bool e4m3) {
    const int G = Hq / Hkv;
    Cut c{};
    const int64_t most = (int64_t)std::max(1, std::min(max_q, T)) * G;  // rows of a sequence
    const int64_t seqs = std::min(S, T), all = (int64_t)T * G;
    const int limit = !e4m3 && most > kFewRows ? kFewRows : 0x7fffffff;
    const bool short_keys = keys <= (int64_t)kWholeSteps * kKeyStep;
    auto plan = [&](int rows, int lo, int hi, int whole_from, int min_steps, Plan& p, int64_t& grid, size_t& bytes) {
        const int64_t rows_each = std::min<int64_t>(most, hi);
        const int64_t tiles = std::min(all / rows + seqs, seqs * ((rows_each + rows - 1) / rows));
        p.rows = rows, p.lo = lo, p.hi = hi;
        p.parts = tiles * Hkv >= whole_from || short_keys ? 0 : std::max(1, kCus / Hkv);
        p.min_steps = min_steps;
        grid = (p.parts ? p.parts : tiles) * Hkv;
        bytes = p.parts ? o_bytes(p, Hkv, D) + ml_bytes(p, Hkv) : 0;
    };
    // (a hint that is too small keeps every sequence in the few-rows kernel; one that is too large costs an idle launch)
    if (!(most > limit && S == 1 && max_q >= T && all > kFewRows))
        plan(std::min<int64_t>(most, limit) <= 16 ? 16 : 32, 1, limit, 8 * kCus, 8, c.few, c.few_grid, c.few_bytes);
    if (most > limit) plan(256, limit + 1, 0x7fffffff, 4 * kCus, 4, c.chunk, c.chunk_grid, c.chunk_bytes);
    return c;
}

inline int64_t most_keys(int width, int page, int causal, int window, int T, int max_q) {
    const int64_t held = (int64_t)width * page;
    return causal && window >= 0 ? std::min(held, (int64_t)window + std::max(1, std::min(max_q, T)) + kKeyStep) : held;
}

template <typename Tag>
int run(const AttnArgs& a, Cut& c, void* ws, int D, bool e4m3, hipStream_t stream) {
    char* at = (char*)ws;
    for (Plan* p : {&c.few, &c.chunk}) {
        p->o = (float*)at;
        at += o_bytes(*p, a.Hkv, D);
        p->ml = (float*)at;
        at += ml_bytes(*p, a.Hkv);
    }
    if (c.chunk.rows)
        if (int rc = launch_chunk<Tag>(a, c.chunk, D, e4m3, c.chunk_grid, stream)) return rc;
    if (c.few.rows)
        if (int rc = launch_few<Tag>(a, c.few, D, e4m3, c.few_grid, stream)) return rc;
    if (c.few.parts || c.chunk.parts) {
        const dim3 grid((unsigned)((int64_t)a.g.T * a.Hq));
        if (D == 128)
            join_kernel<Tag, 128><<<grid, kJoinWaves * 64, 0, stream>>>(a, c.few, c.chunk);
        else
            join_kernel<Tag, 64><<<grid, kJoinWaves * 64, 0, stream>>>(a, c.few, c.chunk);
        return launch_status();
    }
    return VQA_OK;
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
    Cut c = cut_call(T, S, Hq, Hkv, D, max_q, most_keys(width, page, causal, window, T, max_q), e4m3 != 0);
    if (c.few_grid > 0x7fffffff || c.chunk_grid > 0x7fffffff) return VQA_ERR_BAD_SHAPE;
    const size_t bytes = c.few_bytes + c.chunk_bytes;
    if (bytes && ws == nullptr) return VQA_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(ws) % 256) return VQA_ERR_MISALIGNED;
    if (ws_bytes < bytes) return VQA_ERR_WORKSPACE_TOO_SMALL;
    return run<Tag>(a, c, ws, D, e4m3 != 0, stream);
}

}  // namespace paged
}  // namespace vqa

extern "C" {

size_t vqa_paged_attn_workspace_bytes(int T, int S, int Hq, int Hkv, int D, int page, int width, int e4m3, int causal,
                                      int window, int max_q) {
    if (T < 1 || S < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv || page < 1 || width < 1) return 0;
    const vqa::paged::Cut c = vqa::paged::cut_call(
        T, S, Hq, Hkv, D, max_q, vqa::paged::most_keys(width, page, causal, window, T, max_q), e4m3 != 0);
    return c.few_bytes + c.chunk_bytes;
}

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
