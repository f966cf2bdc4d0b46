// Attention of new tokens over the paged cache: arguments, visibility rule, and the plain one-row form that every kernel
// can fall back to.
//
// Row t (0 <= t < n) of a sequence with `len` keys stands at i = len - n + t and sees the keys j that exist (j < keys, their
// page is there) with j <= i and i - j <= window when causal, all of them otherwise.  A row that sees nothing gets 0 and
// lse = -inf.
#pragma once

#include "vqa_paged.h"

namespace vqa {
namespace paged {

struct AttnArgs {
    Pool kp, vp;
    Seqs g;
    const uint16_t* q;
    int64_t q_st, q_sh;  // elements
    uint16_t* out;
    int64_t o_st, o_sh;
    float* lse;  // [T, Hq] contiguous, nullable
    int Hq, Hkv, G;
    int causal, window;  // window: a number no distance reaches where there is none
    float scale_log2e;
};

// keys [lo, hi) that row t of the sequence may see
struct Range {
    int lo, hi;
};
__device__ __forceinline__ Range visible(const AttnArgs& a, const Seq& s, int t) {
    if (!a.causal) return {0, s.keys};
    const int i = s.len - s.n + t;
    return {max(0, i - a.window), min(s.keys, i + 1)};
}

// Unnormalised attention of ONE row over keys [lo, hi), by one wave in fp32: the definition, key by key.  A lane scores one
// key of 64, then the wave adds the weighted value rows one by one, skipping the keys the row does not see -- so what lies
// in hidden places (infinities, NaN, memory never written) is not even multiplied by zero.
template <int D>
struct RowState {
    float m, l;       // same in every lane
    float o[D / 64];  // elements lane * (D / 64) ..
};

template <typename Tag, int D, bool kE4m3>
__device__ __noinline__ void row_by_lanes(const AttnArgs& a, int s, int h, const uint16_t* q, int lo, int hi,
                                          RowState<D>& st, int lane) {
    constexpr int E = D / 64;
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) st.o[e] = 0.f;
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        const int page = j < hi ? page_of(a.g, s, j) : -1;
        float sc = -INFINITY, vf = 0.f;
        const char* v_row = nullptr;
        if (page >= 0) {
            const char* k_row = row_of(a.kp, a.g, page, h, j);
            v_row = row_of(a.vp, a.g, page, h, j);
            float f = 1.f;
            if constexpr (kE4m3) {
                f = factor_of(*exp_of(a.kp, a.g, page, h, j));
                vf = factor_of(*exp_of(a.vp, a.g, page, h, j));
            }
            float dot = 0.f;
            for (int d = 0; d < D; d += 8) {
                const uint4 qw = *reinterpret_cast<const uint4*>(q + d);
                const uint32_t qx[4] = {qw.x, qw.y, qw.z, qw.w};
                uint32_t kx[4];
                if constexpr (kE4m3) {
                    const uint2 w = *reinterpret_cast<const uint2*>(k_row + d);
                    const uint2 p0 = widen4<Tag>(w.x, f), p1 = widen4<Tag>(w.y, f);
                    kx[0] = p0.x, kx[1] = p0.y, kx[2] = p1.x, kx[3] = p1.y;
                } else {
                    const uint4 w = *reinterpret_cast<const uint4*>(k_row + 2 * d);
                    kx[0] = w.x, kx[1] = w.y, kx[2] = w.z, kx[3] = w.w;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dot = __builtin_fmaf(Elem<Tag>::from_bits((uint16_t)(qx[e] & 0xffffu)),
                                         Elem<Tag>::from_bits((uint16_t)(kx[e] & 0xffffu)), dot);
                    dot = __builtin_fmaf(Elem<Tag>::from_bits((uint16_t)(qx[e] >> 16)),
                                         Elem<Tag>::from_bits((uint16_t)(kx[e] >> 16)), dot);
                }
            }
            sc = dot * a.scale_log2e;
        }
        // a visible score of NaN must reach the output: fmaxf drops it, exp2 below does not
        const float m_new = fmaxf(st.m, wave_max(sc));
        const float m_safe = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = fast_exp2(st.m - m_safe);
        const float p = page >= 0 ? fast_exp2(sc - m_safe) : 0.f;
        st.m = m_new;
        st.l = st.l * alpha + wave_sum(p);
#pragma unroll
        for (int e = 0; e < E; ++e) st.o[e] *= alpha;
        uint64_t todo = __builtin_amdgcn_ballot_w64(page >= 0);
        while (todo) {
            const int kk = __builtin_ctzll(todo);
            todo &= todo - 1;
            const float pk = __shfl(p, kk, 64);
            const uint64_t row = (uint64_t)(uintptr_t)v_row;
            const uint32_t r_lo = __shfl((uint32_t)row, kk, 64), r_hi = __shfl((uint32_t)(row >> 32), kk, 64);
            const char* vr = reinterpret_cast<const char*>((uintptr_t)(((uint64_t)r_hi << 32) | r_lo));
            float x[E];
            if constexpr (kE4m3) {
                const float f = __shfl(vf, kk, 64);
                uint32_t w;
                if constexpr (E == 2)
                    w = *reinterpret_cast<const uint16_t*>(vr + lane * 2);
                else
                    w = *reinterpret_cast<const uint8_t*>(vr + lane);
                const uint2 u = widen4<Tag>(w, f);
                x[0] = Elem<Tag>::from_bits((uint16_t)(u.x & 0xffffu));
                if constexpr (E == 2) x[1] = Elem<Tag>::from_bits((uint16_t)(u.x >> 16));
            } else {
                const uint16_t* vw = reinterpret_cast<const uint16_t*>(vr) + lane * E;
                x[0] = Elem<Tag>::from_bits(vw[0]);
                if constexpr (E == 2) x[1] = Elem<Tag>::from_bits(vw[1]);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) st.o[e] = __builtin_fmaf(pk, x[e], st.o[e]);
        }
    }
}

// Normalise and store one row held by a wave as row_by_lanes leaves it.
template <typename Tag, int D>
__device__ __forceinline__ void store_row(const AttnArgs& a, const RowState<D>& st, int row, int hq, int lane) {
    const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
    uint16_t* dst = a.out + (int64_t)row * a.o_st + (int64_t)hq * a.o_sh;
    if constexpr (D == 128) {
        const uint32_t w = (uint32_t)Elem<Tag>::to_bits(st.o[0] * inv) | ((uint32_t)Elem<Tag>::to_bits(st.o[1] * inv) << 16);
        *reinterpret_cast<uint32_t*>(dst + 2 * lane) = w;
    } else {
        dst[lane] = Elem<Tag>::to_bits(st.o[0] * inv);
    }
    if (a.lse != nullptr && lane == 0)
        a.lse[(int64_t)row * a.Hq + hq] = st.l == 0.f ? -INFINITY : st.m + fast_log2(st.l);
}

}  // namespace paged
}  // namespace vqa
