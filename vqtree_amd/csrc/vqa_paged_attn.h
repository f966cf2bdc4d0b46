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
// Work units.  The new rows of a sequence and the G query heads of a key head are one list of n * G rows (row r: new token
// r / G, head r % G of the group), cut into tiles; the keys a sequence's rows see are cut into splits.  A unit is one tile
// and one split of one sequence.  How long a split is follows from the lengths found on the device: the work of the call
// over the number of workgroups that fill the chip, so a batch of unequal lengths is spread evenly and a recorded call
// adapts to new ones.  Every kernel of a call computes the same plan from the same numbers.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kKeyStep = 64;  // splits begin and end at multiples of this many keys

struct Plan {
    int rows;       // rows of a tile
    int lo, hi;     // sequences with lo <= n * G <= hi belong to this kernel
    int max_tiles;  // the grid and the workspace are made for this many tiles (of one key head) ...
    int units;      // ... and units; more of either (a wrong hint): no splits
    int per_head;   // workgroups worth having per key head
    int min_steps;  // shortest split, in key steps
    float* o;       // partial results [unit * Hkv + head][rows][D], unnormalised
    float* ml;      // [..][rows][2]: maximum (base 2, scaled) and sum
};

struct Share {  // what one sequence brings
    int tiles, first, steps;  // row tiles; first key step its rows see; number of key steps
};
__device__ __forceinline__ Share share_of(const AttnArgs& a, const Plan& p, int s) {
    if (s >= a.g.S) return {0, 0, 0};
    const Seq q = seq_of(a.g, s);
    const int64_t rows = (int64_t)q.n * a.G;
    if (rows < 1 || rows < p.lo || rows > p.hi) return {0, 0, 0};
    const Range r0 = visible(a, q, 0);
    const int hi = visible(a, q, q.n - 1).hi;
    Share x;
    x.tiles = (int)((rows + p.rows - 1) / p.rows);
    x.first = r0.lo / kKeyStep;
    x.steps = max(0, (hi + kKeyStep - 1) / kKeyStep - x.first);
    return x;
}

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)x, o, 64), hi = __shfl_xor((uint32_t)(x >> 32), o, 64);
        x += (int64_t)(((uint64_t)hi << 32) | lo);
    }
    return x;
}

// Key steps per split of this call (0x7fffffff: no splits), the same in every wave.
__device__ __forceinline__ int split_steps(const AttnArgs& a, const Plan& p, int lane) {
    int64_t work = 0, tiles = 0;
    for (int base = 0; base < a.g.S; base += kWave) {
        const Share x = share_of(a, p, base + lane);
        work += (int64_t)x.tiles * x.steps;
        tiles += x.tiles;
    }
    work = wave_sum64(work);
    tiles = wave_sum64(tiles);
    if (tiles > p.max_tiles || p.per_head < 1) return 0x7fffffff;
    const int64_t per = (work + p.per_head - 1) / p.per_head;
    // sum over tiles of ceil(steps / per) <= work / per + tiles <= per_head + max_tiles = units
    return (int)max((int64_t)p.min_steps, per < 0x7fffffff ? per : 0x7fffffff);
}
__device__ __forceinline__ int splits_of(const Share& x, int per) {
    return x.steps <= per ? 1 : (x.steps + per - 1) / per;
}

struct Unit {
    int s, tile, split, n_splits, slot;  // slot: number of the unit (its place in the workspace)
    int first, steps;                    // the sequence's key steps
};
// unit x of the call, s = -1 if there is none
__device__ __forceinline__ Unit find_unit(const AttnArgs& a, const Plan& p, int per, int64_t x, int lane) {
    Unit u;
    u.s = -1;
    int64_t before = 0;
    for (int base = 0; base < a.g.S; base += kWave) {
        const Share h = share_of(a, p, base + lane);
        const int n_splits = splits_of(h, per);
        // (tiles * splits of one sequence fits 32 bits: with splits there are at most `units` of them, without it is the
        // number of tiles)
        const int mine = h.tiles * n_splits;
        int64_t sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t lo = __shfl_up((uint32_t)sum, o, 64), hi = __shfl_up((uint32_t)(sum >> 32), o, 64);
            if (lane >= o) sum += (int64_t)(((uint64_t)hi << 32) | lo);
        }
        const bool here = x < before + sum;
        const uint64_t vote = __builtin_amdgcn_ballot_w64(here);
        if (vote) {
            const int at = __builtin_ctzll(vote);
            const int64_t start = before + sum - mine;
            const int64_t rest = x - start;
            u.s = base + at;
            const int local = __shfl((int)rest, at, 64);
            u.n_splits = __shfl(n_splits, at, 64);
            u.first = __shfl(h.first, at, 64);
            u.steps = __shfl(h.steps, at, 64);
            u.tile = local / u.n_splits;
            u.split = local % u.n_splits;
            u.slot = (int)x;
            return u;
        }
        before += wave_sum64(mine);
    }
    return u;
}
// keys [first, last) of a split: the steps are dealt out evenly
__device__ __forceinline__ Range split_keys(const Unit& u) {
    const int a = (int)((int64_t)u.steps * u.split / u.n_splits), b = (int)((int64_t)u.steps * (u.split + 1) / u.n_splits);
    return {(u.first + a) * kKeyStep, (u.first + b) * kKeyStep};
}

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
