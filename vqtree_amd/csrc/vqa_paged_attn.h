// Attention of new tokens over the paged cache: arguments, visibility rule, and the plain one-row form that every kernel
// can fall back to.
//
// Row t (0 <= t < n) of a sequence with `len` keys stands at i = len - n + t and sees the keys j that exist (j < keys, their
// page is there) with j <= i and i - j <= window when causal, all of them otherwise.  A row that sees nothing gets 0 and
// lse = -inf.
#pragma once

#include <mutex>

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
__device__ __forceinline__ void row_by_lanes(const AttnArgs& a, int s, int h, const uint16_t* q, int lo, int hi,
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

// ---------------------------------------------------------------------------------------------------------------------
// Work.  The new rows of a sequence and the G query heads of a key head are one list of n * G rows (row r: new token
// r / G, head r % G of the group), cut into tiles; a tile has as many key steps (64 keys) as its sequence's rows see.  With
// splits, the steps of all tiles of a key head stand in one line and each of its `parts` workgroups takes an equal piece of it,
// wherever tiles begin and end: the lengths are known on the device only, and however unequal they are (and whatever a
// recorded call meets when it is replayed) all workgroups end together.  A piece that is not a whole tile leaves an
// unnormalised result, which join_kernel puts together.  Without splits a workgroup takes whole tiles.
// Every kernel of a call computes the same plan from the same numbers.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kKeyStep = 64;

struct Plan {
    int rows;       // rows of a tile
    int lo, hi;     // sequences with lo <= n * G <= hi belong to this kernel
    int parts;      // workgroups per key head that share the steps; 0: no splits
    int min_steps;  // fewest steps worth a workgroup
    float* o;       // partial results [2 * part + (not the part's first piece)][Hkv][rows][D], unnormalised
    float* ml;      // [..][rows][2]: maximum (base 2, scaled) and sum
};

struct Share {  // what one sequence brings
    int tiles, first, steps;  // row tiles; first key step its rows see; number of steps of a tile
};
__device__ __forceinline__ Share share_of(const AttnArgs& a, const Plan& p, int s) {
    if (s >= a.g.S) return {0, 0, 0};
    const Seq q = seq_of(a.g, s);
    const int64_t rows = (int64_t)q.n * a.G;
    if (rows < 1 || rows < p.lo || rows > p.hi) return {0, 0, 0};
    const int hi = visible(a, q, q.n - 1).hi;
    Share x;
    x.tiles = (int)((rows + p.rows - 1) / p.rows);
    x.first = visible(a, q, 0).lo / kKeyStep;
    x.steps = max(1, (hi + kKeyStep - 1) / kKeyStep - x.first);  // (a tile that sees nothing is still stored)
    return x;
}
__device__ __forceinline__ int64_t weight_of(const Plan& p, const Share& x) {
    return p.parts ? (int64_t)x.tiles * x.steps : x.tiles;
}

__device__ __forceinline__ int64_t lane64(int64_t x, int from) {  // (from: the same in every lane)
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, from);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), from);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t scan64(int64_t x, int lane) {  // sum over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t lo = __shfl_up((uint32_t)x, o, 64), hi = __shfl_up((uint32_t)(x >> 32), o, 64);
        if (lane >= o) x += (int64_t)(((uint64_t)hi << 32) | lo);
    }
    return x;
}

struct Piece {
    int s, tile;      // sequence (-1: none), row tile
    int first, steps; // key steps of the whole tile
    int from;         // of them, where the position lies
};

// The line of work of one key head, held by a wave.
struct Line {
    Share mine;       // of sequence `lane`: batches of up to 64 sequences are read once
    int64_t sum;      // weights of the sequences up to and with that one
    int64_t total;
    int parts;        // workgroups that share it (at most p.parts)

    __device__ __forceinline__ void init(const AttnArgs& a, const Plan& p, int lane) {
        mine = share_of(a, p, lane);
        sum = scan64(weight_of(p, mine), lane);
        total = lane64(sum, 63);
        for (int base = kWave; base < a.g.S; base += kWave)
            total += lane64(scan64(weight_of(p, share_of(a, p, base + lane)), lane), 63);
        parts = 0;
        if (p.parts) parts = (int)max((int64_t)1, min((int64_t)p.parts, total / p.min_steps));
    }
    __device__ __forceinline__ int64_t start(int i) const { return total * i / parts; }            // of part i
    __device__ __forceinline__ int part_of(int64_t x) const { return (int)(((x + 1) * parts - 1) / total); }

    __device__ __forceinline__ Piece find(const AttnArgs& a, const Plan& p, int64_t x, int lane) const {
        Piece r = {-1, 0, 0, 0, 0};
        if (x >= total) return r;
        Share h = mine;
        int64_t upto = sum, before = 0;
        for (int base = 0;;) {
            const uint64_t vote = __builtin_amdgcn_ballot_w64(x < before + upto);
            if (vote) {
                const int at = __builtin_ctzll(vote);
                const int64_t rest = x - lane64(before + upto - weight_of(p, h), at);
                r.s = __builtin_amdgcn_readfirstlane(base + at);
                r.first = __builtin_amdgcn_readlane(h.first, at);
                r.steps = __builtin_amdgcn_readlane(h.steps, at);
                r.tile = __builtin_amdgcn_readfirstlane((int)(p.parts ? rest / r.steps : rest));
                r.from = __builtin_amdgcn_readfirstlane(p.parts ? (int)(rest - (int64_t)r.tile * r.steps) : 0);
                return r;
            }
            before += lane64(upto, 63);
            base += kWave;
            h = share_of(a, p, base + lane);
            upto = scan64(weight_of(p, h), lane);
        }
    }
    // position of the first step of a sequence's first tile (s uniform)
    __device__ __forceinline__ int64_t start_of(const AttnArgs& a, const Plan& p, int s, int lane) const {
        Share h = mine;
        int64_t upto = sum, before = 0;
        for (int base = 0; s >= base + kWave;) {
            before += lane64(upto, 63);
            base += kWave;
            h = share_of(a, p, base + lane);
            upto = scan64(weight_of(p, h), lane);
        }
        return before + lane64(upto - weight_of(p, h), s & 63);
    }
};

// Kernels that use more than 64 KB of LDS need the limit raised once per device: the one that owns the operands.
template <auto kKernel>
int raise_lds(const void* operand, int bytes) {
    static std::mutex mutex;
    static bool raised[kMaxDevices] = {};
    int dev = 0;
    if (int rc = device_of_pointer(operand, &dev)) return rc;
    std::lock_guard<std::mutex> lock(mutex);
    if (!raised[dev]) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
            hipSuccess)
            return VQA_ERR_LAUNCH_FAILED;
        raised[dev] = true;
    }
    return VQA_OK;
}

template <typename Tag>
int launch_few(const AttnArgs& a, const Plan& p, int D, bool e4m3, int64_t grid, hipStream_t stream);

}  // namespace paged
}  // namespace vqa
