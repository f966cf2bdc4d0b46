// The paged key / value cache: how a row is found and what it holds, shared by the kernels that write it, read it back
// and attend over it.
//
// Row j of sequence s lies in page block_table[s][j / page], at place j % page of every head; a pool is
// [pages, Hkv, page, D].  A table entry outside [0, pages) is a page that is not there: nothing is written to it, its rows
// read as zero and its keys are hidden.  Rows come in the element type, or as e4m3 with one byte per row that holds a power of
// two (value = e4m3 * 2^(byte - 127)): a power of two costs the values nothing -- e4m3 has four significant bits wherever a
// row's largest magnitude lies, for that and for everything down to 2^-14 of it (below, its steps stay the same) -- and gfx950 converts with such a factor in the same instruction
// (v_cvt_scalef32_pk_*_fp8), so what the attention multiplies is the stored value exactly, without a scale in the scores.
#pragma once

#include "vqa_common.h"

namespace vqa {
namespace paged {

struct Pool {  // strides in bytes
    char* p;
    int64_t sp, sh, sn;
    uint8_t* e;  // exponent bytes, null in 16 bits
    int64_t ep, eh;
};

struct Seqs {
    const int32_t* cu;     // [S + 1]: new rows of sequence s are the packed rows cu[s] .. cu[s + 1]
    const int32_t* lens;   // [S]: keys of a sequence, its new rows included
    const int32_t* table;  // [S, width]
    int64_t table_ss;
    int S, T, width, n_pages, page_shift;
};

// What the device reads is data and may be anything: every number that ends up in an address is brought into range here.
struct Seq {
    int q0, n;     // first packed row, number of new rows
    int len;       // keys according to kv_lens, at least 0
    int keys;      // keys the table can hold of them
};
__device__ __forceinline__ Seq seq_of(const Seqs& g, int s) {
    Seq r;
    r.q0 = min(max(g.cu[s], 0), g.T);
    r.n = min(max(g.cu[s + 1], r.q0), g.T) - r.q0;
    r.len = max(g.lens[s], 0);
    r.keys = min(r.len, g.width << g.page_shift);
    return r;
}

// page of row j (0 <= j < width << page_shift) of sequence s, -1 if it is not there
__device__ __forceinline__ int page_of(const Seqs& g, int s, int j) {
    const int page = g.table[(int64_t)s * g.table_ss + (j >> g.page_shift)];
    return (unsigned)page < (unsigned)g.n_pages ? page : -1;
}

__device__ __forceinline__ char* row_of(const Pool& pool, const Seqs& g, int page, int h, int j) {
    return pool.p + (int64_t)page * pool.sp + (int64_t)h * pool.sh + (int64_t)(j & ((1 << g.page_shift) - 1)) * pool.sn;
}
__device__ __forceinline__ uint8_t* exp_of(const Pool& pool, const Seqs& g, int page, int h, int j) {
    return pool.e + (int64_t)page * pool.ep + (int64_t)h * pool.eh + (j & ((1 << g.page_shift) - 1));
}

// 2^(byte - 127); byte 0 (never written by the quantiser) counts as 2^-126
__device__ __forceinline__ float factor_of(int byte) {
    return __builtin_bit_cast(float, (uint32_t)max(byte, 1) << 23);
}

// four e4m3 values times a power of two, as two packed pairs of the element type: exact in bf16 (4 significant bits); in f16
// exact down to its subnormal numbers, where the last place is rounded
template <typename Tag>
__device__ __forceinline__ uint2 widen4(uint32_t x, float factor);
template <>
__device__ __forceinline__ uint2 widen4<bf16_tag>(uint32_t x, float factor) {
    const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, factor, false);
    const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, factor, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}
template <>
__device__ __forceinline__ uint2 widen4<f16_tag>(uint32_t x, float factor) {
    const f16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, factor, false);
    const f16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, factor, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// ---------------------------------------------------------------------------------------------------------------------
// Host side: what every entry point checks of the cache's description before its first launch.
// ---------------------------------------------------------------------------------------------------------------------
inline bool pow2(int x) { return x > 0 && (x & (x - 1)) == 0; }

// strides: pages (p, h, n) in elements, exponents (p, h)
inline int make_pool(Pool* pool, const void* pages, const uint8_t* exps, const int64_t* s, const int64_t* es, int e4m3,
                     int page) {
    const int64_t size = e4m3 ? 1 : 2;
    if (pages == nullptr || (e4m3 && exps == nullptr)) return VQA_ERR_NULL_POINTER;
    *pool = Pool{(char*)pages, s[0] * size, s[1] * size, s[2] * size, e4m3 ? (uint8_t*)exps : nullptr, e4m3 ? es[0] : 0,
                 e4m3 ? es[1] : 0};
    // (the exponents of 16 rows are fetched as one piece)
    if (e4m3 && (!aligned16(exps) || es[0] % 16 || es[1] % 16 || es[0] < 0 || es[0] >= (int64_t(1) << 32)))
        return VQA_ERR_MISALIGNED;
    if (!aligned16(pages) || pool->sp % 16 || pool->sh % 16 || pool->sn % 16) return VQA_ERR_MISALIGNED;
    // a row's offset inside its page is kept in 32 bits
    if (pool->sn < 0 || pool->sn * page >= (int64_t(1) << 31)) return VQA_ERR_MISALIGNED;
    return VQA_OK;
}

inline int make_seqs(Seqs* g, const int32_t* cu, const int32_t* lens, const int32_t* table, int64_t table_ss, int S, int T,
                     int width, int n_pages, int page) {
    if (S < 0 || T < 0 || width < 1 || n_pages < 1) return VQA_ERR_BAD_SHAPE;
    if (!pow2(page) || page < 16 || page > 4096) return VQA_ERR_BAD_ARGUMENT;
    if ((int64_t)width * page > (int64_t(1) << 30)) return VQA_ERR_BAD_SHAPE;
    *g = Seqs{cu, lens, table, table_ss, S, T, width, n_pages, __builtin_ctz(page)};
    return VQA_OK;
}

}  // namespace paged
}  // namespace vqa
