// Attention of new tokens over the paged cache (vqa_paged_attn_*).
#include <algorithm>

#include "vqa_paged_attn.h"

namespace vqa {
namespace paged {

// Joins the pieces of a tile: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.  A tile in pieces holds the place where
// some part begins, and the first such part has noted it; the rows of all noted tiles are dealt out to the waves.  What it
// costs is latency -- partial results come from other XCDs' caches or from HBM, 1 - 2 us a round -- so a wave asks for kAhead
// pieces of kRowsEach rows at once.
constexpr int kJoinWaves = 8;

template <typename Tag, int D>
__global__ __launch_bounds__(kJoinWaves * 64) void join_kernel(AttnArgs a, Plan few, Plan chunk) {
    constexpr int E = D / 64;
    constexpr int kAhead = 8, kRowsEach = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Plan& p = few.parts == 0 || blockIdx.z ? chunk : few;
    const int n_notes = p.parts * a.Hkv;
    int64_t item = (int64_t)blockIdx.x * kJoinWaves + wave;  // number of the group of rows among all groups to join
    int64_t before = 0;
    for (int base4 = 0; base4 < n_notes; base4 += 256) {
    // (the notes of up to 256 parts are asked for at once: there are no more where a part is a compute unit)
    int4 notes[4];
    int2 more[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int* src = p.joins + (int64_t)min(base4 + b * 64 + lane, n_notes - 1) * kJoinInts;
        notes[b] = *reinterpret_cast<const int4*>(src);
        more[b] = *reinterpret_cast<const int2*>(src + 4);
        if (base4 + b * 64 + lane >= n_notes) notes[b].x = 0;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int base = base4 + b * 64;
        const int4 d = notes[b];
        const int2 d2 = more[b];
        const int mine = d.x ? (d.w + kRowsEach - 1) / kRowsEach : 0;
        const int upto = scan32(mine);
        const int64_t here = __builtin_amdgcn_readlane(upto, 63);
        for (; item < before + here; item += (int64_t)gridDim.x * kJoinWaves) {
            const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(item < before + upto));
            // rows r0 .. of the tile
            const int r0 = ((int)(item - before) - __builtin_amdgcn_readlane(upto - mine, at)) * kRowsEach;
            const int n = __builtin_amdgcn_readlane(d.x, at), q0 = __builtin_amdgcn_readlane(d.y, at);
            const int row0 = __builtin_amdgcn_readlane(d.z, at), n_rows = __builtin_amdgcn_readlane(d.w, at);
            const int i0 = __builtin_amdgcn_readlane(d2.x, at), shift = __builtin_amdgcn_readlane(d2.y, at);
            const int h = (base + at) % a.Hkv;
            // piece k lies with part i0 + k; that of part i0 itself may be its second
            const int64_t step = (int64_t)2 * a.Hkv * p.rows, skew = (int64_t)shift * a.Hkv * p.rows;
            const int64_t first = (int64_t)i0 * step + (int64_t)h * p.rows;
            auto place = [&](int k, int r) { return first + k * step + (k ? 0 : skew) + min(r0 + r, n_rows - 1); };
            // lane 8 * r + k weighs piece k of row r (lanes from 32 on repeat those)
            const int my_k = lane % kAhead, my_r = lane / kAhead % kRowsEach;
            float m_run = -INFINITY, l_run = 0.f, o[kRowsEach][E];
#pragma unroll
            for (int r = 0; r < kRowsEach; ++r)
#pragma unroll
                for (int e = 0; e < E; ++e) o[r][e] = 0.f;
            for (int k0 = 0; k0 < n; k0 += kAhead) {
                const int k = k0 + my_k;
                const float2 ml = *reinterpret_cast<const float2*>(p.ml + place(min(k, n - 1), my_r) * 2);
                float x[kAhead][kRowsEach][E];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
#pragma unroll
                    for (int r = 0; r < kRowsEach; ++r)
#pragma unroll
                        for (int e = 0; e < E; ++e) x[j][r][e] = 0.f;
                    if (k0 + j < n) {  // (uniform)
#pragma unroll
                        for (int r = 0; r < kRowsEach; ++r)
#pragma unroll
                            for (int e = 0; e < E; ++e) x[j][r][e] = p.o[place(k0 + j, r) * D + lane * E + e];
                    }
                }
                const float m = k < n ? ml.x : -INFINITY;
                float top = m;
#pragma unroll
                for (int s = 1; s < kAhead; s <<= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
                top = fmaxf(top, m_run);
                const float ref = top == -INFINITY ? 0.f : top;
                const float alpha = fast_exp2(m_run - ref), f = fast_exp2(m - ref);
                float l = k < n ? f * ml.y : 0.f;
#pragma unroll
                for (int s = 1; s < kAhead; s <<= 1) l += __shfl_xor(l, s, 64);
                l_run = l_run * alpha + l;
                m_run = top;
#pragma unroll
                for (int r = 0; r < kRowsEach; ++r) {
                    const float al = __shfl(alpha, r * kAhead, 64);
#pragma unroll
                    for (int e = 0; e < E; ++e) o[r][e] *= al;
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) {
                        const float w = __shfl(f, r * kAhead + j, 64);
#pragma unroll
                        for (int e = 0; e < E; ++e) o[r][e] += w * x[j][r][e];
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < kRowsEach; ++r) {
                if (r0 + r >= n_rows) continue;
                RowState<D> st;
                st.m = __shfl(m_run, r * kAhead, 64), st.l = __shfl(l_run, r * kAhead, 64);
#pragma unroll
                for (int e = 0; e < E; ++e) st.o[e] = o[r][e];
                const int rr = row0 + r0 + r, t = rr / a.G;
                store_row<Tag, D>(a, st, q0 + t, h * a.G + rr - t * a.G, lane);
            }
        }
        before += here;
    }
    }
}

// How a call is cut up (host side; how many rows and keys there are is known on the device only).
struct Cut {
    Plan few, chunk;                // (a plan without rows: its kernel is not needed)
    int64_t few_grid, chunk_grid;
    size_t few_bytes, chunk_bytes;  // workspace
};

constexpr int kCus = 256;           // workgroups that fill the chip: one per compute unit, in both kernels

// A tile of so few key steps is not worth a split and the launch that joins it: one token, 32 query and 8 key heads, whole /
// split: 12.7 / 16.2 us for 1020 keys, 17.5 / 16.4 for 2000, 26.4 / 18.3 for 4000.  (Chunks of 2048 rows over 1500 keys: 53 /
// 59.)
constexpr int kWholeSteps = 32;

// Sequences of more rows than this go to the chunk kernel, which reads the keys once for 256 rows where the few-rows kernel
// does for 32, at a higher rate of products, but starts and ends slower: few / chunk, 32 new tokens for 4 x 8 heads (128 rows):
// 32 sequences of 4096 keys 221 / 192 us, 8 of 2000 to 8300 keys 101 / 75; 16 new tokens (64 rows), one sequence of 4096 or
// 32768 keys 21 / 29, 38 / 58.  Calls with little to do stay in the few-rows kernel: tiles of 32 rows x key heads x (keys, as far
// as the host knows them -- what the table has room for, or the window -- and kTileKeys for the ends of a tile) below kSmall.  1024 rows x 1500 keys (0.5 M): 23 / 52; 256 rows,
// 8 sequences of 160 to 510 keys, and 512 of 230 to 580 (0.6, 1.1 M): 21 / 43, 33 / 41; 20 to 230 rows of 21 sequences and 12
// heads, window 77 (0.8 M): 32 / 52; 2048 rows x 1500 keys (1.0 M): 32 / 53; 128 rows x 32768 keys (1.1 M): 51 / 60; 2 sequences
// of 7 x 1150 rows and 5 heads, window 51 (1.6 M): 54 / 52; 256 rows x 32768 keys (2.1 M): 83 / 65; 1024 rows, 8 sequences of 360
// to 710 keys (2.5 M): 68 / 47; 26000 rows in 7 sequences and 5 heads, window 91 (2.8 M): 75 / 58.
constexpr int kFewRows = 64;
constexpr double kSmall = 3 << 19;
constexpr int kTileKeys = 512;

// The few-rows kernel's tiles have 16 rows where that is all there are (one token / 16 sequences of it, 4 x 8 heads, 16 rows
// against 32: 12.9 / 15.8, 193 / 223 us), and where a workgroup is left for each of them and little to read twice: 20 rows of 8
// sequences 12.1 / 14.4, 64 rows of 8 short sequences 13.8 / 17.0, 512 rows x 128 keys 9.4 / 11.5, x 1500 keys 17.6 / 21.2; but
// 1024 rows x 256 keys (512 tiles of 16) 17.2 / 12.2, 64 rows x 32768 keys 54 / 38, 32 sequences of 64 rows x 4096 222 / 118.
constexpr double kSmall16 = 1 << 19;

// So many tiles are taken whole, one to a workgroup in the order of the grid, without a plan's search or a join.  Few rows: 512
// tiles of 100 to 8000 keys are 181 us whole and 174 dealt out, 1024: 335 and 325, 2048: 637 and 639.  Chunks: between 1 and 8
// times the compute units the time is the same within 3 %, as the plan takes tiles whole by itself where that is best.
constexpr int kWholeTilesFew = 8 * kCus, kWholeTilesChunk = 4 * kCus;

// Workgroups of the few-rows kernel have 8 waves; 4, two to a compute unit, where whole tiles are more than the units.  43
// sequences of 16 to 855 keys, 32 heads: 54 / 69 us with 4 / 8 waves, e4m3 and head dim 64 34 / 52; 403 tokens of 4 x 8 heads
// 13.4 / 22; 16 sequences up to 32 768 keys 192 / 193, but one sequence of 1000 keys 15.8 / 12.9, 65 536 in e4m3 126 / 97.
constexpr int kManyWaves = 8, kFewWaves = 4;

inline size_t round256(size_t x) { return (x + 255) & ~size_t(255); }
inline size_t o_bytes(const Plan& p, int Hkv, int D) { return round256((size_t)2 * p.parts * Hkv * p.rows * D * 4); }
inline size_t join_bytes(const Plan& p, int Hkv) { return round256((size_t)p.parts * Hkv * kJoinInts * 4); }
inline size_t ml_bytes(const Plan& p, int Hkv) { return round256((size_t)2 * p.parts * Hkv * p.rows * 8); }

inline Cut cut_call(int T, int S, int Hq, int Hkv, int D, int page, int width, int causal, int window, int max_q) {
    const int G = Hq / Hkv;
    Cut c{};
    const int64_t most = (int64_t)std::max(1, std::min(max_q, T)) * G;  // rows of a sequence
    const int64_t seqs = std::min(S, T), all = (int64_t)T * G;
    auto tiles_of = [&](int rows, int64_t rows_each) {  // at most, over all sequences
        return std::min(all / rows + seqs, seqs * ((rows_each + rows - 1) / rows));
    };
    // most keys a tile can see, as far as the caller's numbers tell
    auto keys_of = [&](int rows) {
        const int64_t held = (int64_t)width * page;
        return causal && window >= 0 ? std::min(held, (int64_t)window + (rows - 1) / G + 2 + kKeyStep) : held;
    };
    const int limit = most <= kFewRows || (double)tiles_of(32, most) * Hkv * (keys_of(32) + kTileKeys) < kSmall ? 0x7fffffff : kFewRows;
    auto plan = [&](int rows, int lo, int hi, int whole_from, Plan& p, int64_t& grid, size_t& bytes) {
        const int64_t tiles = tiles_of(rows, std::min<int64_t>(most, hi));
        p.rows = rows, p.lo = lo, p.hi = hi;
        const bool short_keys = keys_of(rows) <= (int64_t)kWholeSteps * kKeyStep;
        p.parts = tiles * Hkv >= whole_from || short_keys ? 0 : std::max(1, kCus / Hkv);
        grid = (p.parts ? p.parts : tiles) * Hkv;
        bytes = o_bytes(p, Hkv, D) + ml_bytes(p, Hkv) + join_bytes(p, Hkv);
    };
    // A hint that is too small keeps every sequence in the few-rows kernel; one that is too large costs an idle launch.  One
    // sequence that may bring as many rows as the call has room for goes to the chunk kernel alone, however few it brings: how
    // many there are only the device knows.
    const bool chunk_alone = most > limit && S == 1 && max_q >= T && all > kFewRows;
    if (!chunk_alone) {
        const int64_t rows_each = std::min<int64_t>(most, limit), tiles16 = tiles_of(16, rows_each);
        const bool rows16 = rows_each <= 16 || (tiles16 * Hkv <= kCus && (double)tiles16 * Hkv * keys_of(16) < kSmall16);
        plan(rows16 ? 16 : 32, 1, limit, kWholeTilesFew, c.few, c.few_grid, c.few_bytes);
        c.few.waves = c.few.parts == 0 && c.few_grid > kCus ? kFewWaves : kManyWaves;
    }
    if (most > limit) plan(256, chunk_alone ? 1 : limit + 1, 0x7fffffff, kWholeTilesChunk, c.chunk, c.chunk_grid, c.chunk_bytes);
    // In key steps of about 1 us (few rows) and 2 us (chunks).  Equal pieces beside the line, chunks: 2048 rows x 4096 keys 62 us
    // with and 74 without, 32 sequences of 128 rows x 4096 keys 177 and 191; no difference where all units are busy anyway, and
    // none for few rows.
    c.few.min_steps = 8, c.few.piece_cost = 2, c.few.join_cost = 2, c.few.even = 0;
    c.chunk.min_steps = 4, c.chunk.piece_cost = 8, c.chunk.join_cost = 10, c.chunk.even = 1;
    return c;
}

template <typename Tag>
int run(const AttnArgs& a, Cut& c, void* ws, int D, bool e4m3, int dev, hipStream_t stream) {
    char* at = (char*)ws;
    for (Plan* p : {&c.few, &c.chunk}) {
        p->o = (float*)at;
        at += o_bytes(*p, a.Hkv, D);
        p->ml = (float*)at;
        at += ml_bytes(*p, a.Hkv);
        p->joins = (int*)at;
        at += join_bytes(*p, a.Hkv);
    }
    if (c.chunk.rows)
        if (int rc = launch_chunk<Tag>(a, c.chunk, D, e4m3, c.chunk_grid, dev, stream)) return rc;
    if (c.few.rows)
        if (int rc = launch_few<Tag>(a, c.few, D, e4m3, c.few_grid, dev, stream)) return rc;
    if (c.few.parts || c.chunk.parts) {
        const dim3 grid(c.chunk.parts ? 2 * kCus : kCus, 1, c.few.parts && c.chunk.parts ? 2 : 1);
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
    if (!(scale > 0.f) || !(scale < 2e38f)) return VQA_ERR_BAD_ARGUMENT;  // (times log2(e) it has to stay finite)
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
    a.window = window < 0 ? 0x7fffffff : window;
    a.scale_log2e = scale * kLog2e;
    if (S == 0 || T == 0) return VQA_OK;
    Cut c = cut_call(T, S, Hq, Hkv, D, page, width, causal, window, max_q);
    if (c.few_grid > 0x7fffffff || c.chunk_grid > 0x7fffffff) return VQA_ERR_BAD_SHAPE;
    const size_t bytes = c.few_bytes + c.chunk_bytes;
    if (bytes && ws == nullptr) return VQA_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(ws) % 256) return VQA_ERR_MISALIGNED;
    if (ws_bytes < bytes) return VQA_ERR_WORKSPACE_TOO_SMALL;
    int dev = 0;
    if (int rc = device_of_pointer(q, &dev)) return rc;
    return run<Tag>(a, c, ws, D, e4m3 != 0, dev, stream);
}

}  // namespace paged
}  // namespace vqa

extern "C" {

size_t vqa_paged_attn_workspace_bytes(int T, int S, int Hq, int Hkv, int D, int page, int width, int e4m3, int causal,
                                      int window, int max_q) {
    if (T < 1 || S < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv || page < 1 || width < 1) return 0;
    const vqa::paged::Cut c = vqa::paged::cut_call(T, S, Hq, Hkv, D, page, width, causal, window, max_q);
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
