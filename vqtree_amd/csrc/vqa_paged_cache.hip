// Writing new rows into the paged cache (vqa_paged_write_*) and reading it back as plain tensors (vqa_paged_read_*).
//
// Both move bytes; MI355X copies large tensors at 4.84 TB/s (read and written) and reads them at about 7 TB/s.
//   Writing, a lane holds 16 elements of a row (8 lanes a row at head dim 128): with 8, which makes every load one contiguous
// kilobyte, the quantiser's instructions per byte cost more than the loads gain (53 against 43 us for 8192 rows of 32 heads, keys
// and values, in a loop over one input).  Workgroups go over the heads first (43 -> 40 us), stores past the caches (47 -> 44 us
// in a loop over several inputs: 4.6 TB/s).  16-bit pages: 56 us for 268 MB, 4.8 TB/s.
//   Reading, a lane holds 8 elements, so that a wave stores contiguous kilobytes, and past the caches: 756 MB in 134 us,
// 5.6 TB/s (in a loop over one input 105 us; 149 with ordinary stores, 214 with 16 elements per lane).  16-bit pages:
// 971 MB in 167 us, 5.8 TB/s.
//
// 8-bit rows.  The factor of a row is the smallest power of two 2^e with max |x| <= 448 * 2^e, 448 being the largest e4m3
// number, so nothing saturates; the quotient is exact in fp32 and is rounded once, to the nearest e4m3 number (ties to even).
// A value and its stored form differ by at most 2^-4 of the value, or 2^(e - 10) where that is more.  Magnitudes beyond
// 1.875 * 2^15 (f16) and 1.875 * 2^127 (bf16) are stored as that: the next e4m3 number would read back as infinity.
// Infinities are stored as it too, NaN as NaN.
#include "vqa_paged.h"

namespace vqa {
namespace paged {

struct WriteArgs {
    const uint16_t *k, *v;
    int64_t k_st, k_sh, v_st, v_sh;  // elements
    Pool kp, vp;
    Seqs g;
    int H;
};

constexpr int kWriteWaves = 4;

// 16 elements of one row, 32 bytes
struct Piece {
    uint4 a, b;
};

template <typename Tag>
__device__ __forceinline__ void store_piece(const Pool& pool, const Seqs& g, const Piece& x, int page, int h, int j,
                                            int piece, bool live, int lanes_per_row) {
    if (pool.e == nullptr) {  // (uniform)
        if (live) {
            char* dst = row_of(pool, g, page, h, j) + piece * 32;
            store_stream16(dst, x.a);
            store_stream16(dst + 16, x.b);
        }
        return;
    }
    constexpr bool kF16 = std::is_same<Tag, f16_tag>::value;
    const float top = kF16 ? 61440.f : __builtin_bit_cast(float, 0x7f700000u);  // 1.875 * 2^15, 1.875 * 2^127
    const uint32_t w[8] = {x.a.x, x.a.y, x.a.z, x.a.w, x.b.x, x.b.y, x.b.z, x.b.w};
    float f[16], most = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float y = Elem<Tag>::from_bits((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
        f[i] = y != y ? y : fminf(fmaxf(y, -top), top);
        most = fmaxf(most, fabsf(f[i]));  // (ignores NaN)
    }
    for (int o = 1; o < lanes_per_row; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    const uint32_t bits = __builtin_bit_cast(uint32_t, most);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);  // mantissa above 1.75: one up
    e = min(max(e, -126), 120);
    const float inv = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i] * inv, f[4 * i + 1] * inv, 0, false);
        out[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2] * inv, f[4 * i + 3] * inv, r, true);
    }
    if (live) {
        store_stream16(row_of(pool, g, page, h, j) + piece * 16, make_uint4(out[0], out[1], out[2], out[3]));
        if (piece == 0) *exp_of(pool, g, page, h, j) = (uint8_t)(e + 127);
    }
}

// One wave: 64 / (D / 16) consecutive packed rows of one head, keys and values.
template <typename Tag, int D>
__global__ __launch_bounds__(kWriteWaves * 64) void write_kernel(WriteArgs a) {
    constexpr int kLanes = D / 16, kRows = 64 / kLanes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // heads first: the heads of a token lie next to each other in the input (head by head, the other order, each workgroup
    // in flight reads another row of a wide matrix)
    const int h = (int)(blockIdx.x % (unsigned)a.H);
    const int t0 = ((int)(blockIdx.x / (unsigned)a.H) * kWriteWaves + wave) * kRows;
    if (t0 >= a.g.T) return;
    const int mine = lane / kLanes, piece = lane % kLanes;
    const int t = t0 + mine;
    const int tc = min(t, a.g.T - 1);
    // the rows are on their way while the sequence is looked up
    const uint4* ks = reinterpret_cast<const uint4*>(a.k + (int64_t)tc * a.k_st + (int64_t)h * a.k_sh) + piece * 2;
    const uint4* vs = reinterpret_cast<const uint4*>(a.v + (int64_t)tc * a.v_st + (int64_t)h * a.v_sh) + piece * 2;
    const Piece kx = {ks[0], ks[1]}, vx = {vs[0], vs[1]};
    // sequence of each of the wave's rows: how many sequences end at or before it (cu is read once for all of them)
    int s = 0;
    for (int base = 0; base < a.g.S; base += kWave) {
        const int i = base + lane;
        const int end = i < a.g.S ? a.g.cu[i + 1] : 0x7fffffff;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int c = __popcll(__builtin_amdgcn_ballot_w64(end <= t0 + r));
            s += r == mine ? c : 0;
        }
    }
    bool live = t < a.g.T && s < a.g.S;
    int page = -1, j = 0;
    if (live) {
        const Seq q = seq_of(a.g, s);
        j = q.len - q.n + (t - q.q0);
        live = t >= q.q0 && t < q.q0 + q.n && j >= 0 && j < (a.g.width << a.g.page_shift);
        if (live) page = page_of(a.g, s, j);
        live = page >= 0;
    }
    store_piece<Tag>(a.kp, a.g, kx, page, h, j, piece, live, kLanes);
    store_piece<Tag>(a.vp, a.g, vx, page, h, j, piece, live, kLanes);
}

struct ReadArgs {
    Pool kp, vp;
    Seqs g;
    uint16_t *k, *v;
    int64_t k_ss, k_sh, k_sn, v_ss, v_sh, v_sn;  // elements
    int n;
};

constexpr int kReadWaves = 4;
constexpr int kReadRounds = 2;  // row groups of a wave, keys and values each: four loads in flight per lane

// One wave: kReadRounds groups of 64 / (D / 8) consecutive rows of one head of one sequence, keys and values.  A lane holds 8
// elements, so every store of a wave is one contiguous kilobyte.
template <typename Tag, int D, bool kE4m3>
__global__ __launch_bounds__(kReadWaves * 64) void read_kernel(ReadArgs a) {
    constexpr int kLanes = D / 8, kRows = 64 / kLanes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = blockIdx.y, s = blockIdx.z;
    const int j0 = (blockIdx.x * kReadWaves + wave) * kRows * kReadRounds + lane / kLanes, piece = lane % kLanes;
    const int keys = min(max(a.g.lens[s], 0), a.g.width << a.g.page_shift);
    typedef typename std::conditional<kE4m3, uint2, uint4>::type Word;
    Word k[kReadRounds], v[kReadRounds];
    int ke[kReadRounds], ve[kReadRounds];
#pragma unroll
    for (int i = 0; i < kReadRounds; ++i) {
        const int j = j0 + i * kRows;
        k[i] = v[i] = Word{};
        ke[i] = ve[i] = 0;
        const int page = j < min(keys, a.n) ? page_of(a.g, s, j) : -1;
        if (page >= 0) {
            const char *kr = row_of(a.kp, a.g, page, h, j), *vr = row_of(a.vp, a.g, page, h, j);
            if constexpr (kE4m3) {
                k[i] = *reinterpret_cast<const uint2*>(kr + piece * 8);
                v[i] = *reinterpret_cast<const uint2*>(vr + piece * 8);
                ke[i] = *exp_of(a.kp, a.g, page, h, j);
                ve[i] = *exp_of(a.vp, a.g, page, h, j);
            } else {
                k[i] = load_stream16(kr + piece * 16);
                v[i] = load_stream16(vr + piece * 16);
            }
        }
    }
    auto wide = [](Word w, int e) {
        if constexpr (kE4m3) {
            const float f = factor_of(e);
            const uint2 x = widen4<Tag>(w.x, f), y = widen4<Tag>(w.y, f);
            return make_uint4(x.x, x.y, y.x, y.y);
        } else {
            return w;
        }
    };
#pragma unroll
    for (int i = 0; i < kReadRounds; ++i) {
        const int j = j0 + i * kRows;
        if (j >= a.n) break;
        store_stream16(a.k + s * a.k_ss + h * a.k_sh + j * a.k_sn + piece * 8, wide(k[i], ke[i]));
        store_stream16(a.v + s * a.v_ss + h * a.v_sh + j * a.v_sn + piece * 8, wide(v[i], ve[i]));
    }
}

template <typename Tag>
int write(const void* k, const void* v, void* k_pages, void* v_pages, uint8_t* k_exp, uint8_t* v_exp,
          const int32_t* table, const int32_t* cu, const int32_t* lens, int T, int S, int H, int D, int page, int n_pages,
          int width, int e4m3, const int64_t* st, hipStream_t stream) {
    if (!k || !v || !k_pages || !v_pages || !table || !cu || !lens || !st) return VQA_ERR_NULL_POINTER;
    if (H < 1 || H > 65535) return VQA_ERR_BAD_SHAPE;
    if (D != 64 && D != 128) return VQA_ERR_UNSUPPORTED_HEAD_DIM;
    WriteArgs a{(const uint16_t*)k, (const uint16_t*)v, st[0], st[1], st[2], st[3], {}, {}, {}, H};
    if (int rc = make_seqs(&a.g, cu, lens, table, st[14], S, T, width, n_pages, page)) return rc;
    if (int rc = make_pool(&a.kp, k_pages, k_exp, st + 4, st + 10, e4m3, page)) return rc;
    if (int rc = make_pool(&a.vp, v_pages, v_exp, st + 7, st + 12, e4m3, page)) return rc;
    if (!aligned16(k) || !aligned16(v) || (st[0] | st[1] | st[2] | st[3]) % 8) return VQA_ERR_MISALIGNED;
    if (S == 0 || T == 0) return VQA_OK;
    const int rows = kWriteWaves * 64 / (D / 16);
    const int64_t blocks = (int64_t)((T + rows - 1) / rows) * H;
    if (blocks > 0x7fffffff) return VQA_ERR_BAD_SHAPE;
    int dev = 0;
    if (int rc = device_of_pointer(k, &dev)) return rc;
    const dim3 grid((unsigned)blocks);
    if (D == 128)
        write_kernel<Tag, 128><<<grid, kWriteWaves * 64, 0, stream>>>(a);
    else
        write_kernel<Tag, 64><<<grid, kWriteWaves * 64, 0, stream>>>(a);
    return launch_status();
}

template <typename Tag>
int read(const void* k_pages, const void* v_pages, const uint8_t* k_exp, const uint8_t* v_exp, const int32_t* table,
         const int32_t* lens, void* k, void* v, int S, int H, int n, int D, int page, int n_pages, int width, int e4m3,
         const int64_t* st, hipStream_t stream) {
    if (!k || !v || !k_pages || !v_pages || !table || !lens || !st) return VQA_ERR_NULL_POINTER;
    if (H < 1 || H > 65535 || S > 65535 || n < 0 || n > (1 << 30)) return VQA_ERR_BAD_SHAPE;
    if (D != 64 && D != 128) return VQA_ERR_UNSUPPORTED_HEAD_DIM;
    ReadArgs a{{}, {}, {}, (uint16_t*)k, (uint16_t*)v, st[11], st[12], st[13], st[14], st[15], st[16], n};
    if (int rc = make_seqs(&a.g, nullptr, lens, table, st[10], S, 0, width, n_pages, page)) return rc;
    if (int rc = make_pool(&a.kp, k_pages, k_exp, st, st + 6, e4m3, page)) return rc;
    if (int rc = make_pool(&a.vp, v_pages, v_exp, st + 3, st + 8, e4m3, page)) return rc;
    if (!aligned16(k) || !aligned16(v) || (st[11] | st[12] | st[13] | st[14] | st[15] | st[16]) % 8)
        return VQA_ERR_MISALIGNED;
    if (S == 0 || n == 0) return VQA_OK;
    int dev = 0;
    if (int rc = device_of_pointer(k, &dev)) return rc;
    const int rows = kReadWaves * kReadRounds * 64 / (D / 8);
    const dim3 grid((n + rows - 1) / rows, H, S);
    if (D == 128 && e4m3)
        read_kernel<Tag, 128, true><<<grid, kReadWaves * 64, 0, stream>>>(a);
    else if (D == 128)
        read_kernel<Tag, 128, false><<<grid, kReadWaves * 64, 0, stream>>>(a);
    else if (e4m3)
        read_kernel<Tag, 64, true><<<grid, kReadWaves * 64, 0, stream>>>(a);
    else
        read_kernel<Tag, 64, false><<<grid, kReadWaves * 64, 0, stream>>>(a);
    return launch_status();
}

}  // namespace paged
}  // namespace vqa

extern "C" {

#define VQA_PAGED_CACHE(sfx, tag)                                                                                        \
    int vqa_paged_write_##sfx(const void* k, const void* v, void* k_pages, void* v_pages, uint8_t* k_exp, uint8_t* v_exp, \
                              const int32_t* block_table, const int32_t* cu_q, const int32_t* kv_lens, int T, int S,      \
                              int H, int D, int page, int n_pages, int width, int e4m3, const int64_t* strides,           \
                              vqa_stream_t stream) {                                                                      \
        return vqa::paged::write<vqa::tag>(k, v, k_pages, v_pages, k_exp, v_exp, block_table, cu_q, kv_lens, T, S, H, D,  \
                                           page, n_pages, width, e4m3, strides, stream);                                  \
    }                                                                                                                     \
    int vqa_paged_read_##sfx(const void* k_pages, const void* v_pages, const uint8_t* k_exp, const uint8_t* v_exp,        \
                             const int32_t* block_table, const int32_t* kv_lens, void* k, void* v, int S, int H, int n,   \
                             int D, int page, int n_pages, int width, int e4m3, const int64_t* strides,                   \
                             vqa_stream_t stream) {                                                                       \
        return vqa::paged::read<vqa::tag>(k_pages, v_pages, k_exp, v_exp, block_table, kv_lens, k, v, S, H, n, D, page,   \
                                          n_pages, width, e4m3, strides, stream);                                         \
    }

VQA_PAGED_CACHE(bf16, bf16_tag)
VQA_PAGED_CACHE(f16, f16_tag)

}  // extern "C"
