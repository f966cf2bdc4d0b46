// Attention of new tokens over the paged cache: arguments, visibility rule, and the plain one-row form that every kernel
// can fall back to.
//
// Row t (0 <= t < n) of a sequence with `len` keys stands at i = len - n + t and sees the keys j that exist (j < keys, their
// page is there) with j <= i and i - j <= window when causal, all of them otherwise.  A row that sees nothing gets 0 and
// lse = -inf.
#pragma once

#include <atomic>
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
    int causal, window;  // window: the largest int, which no distance reaches, where there is none
    float scale_log2e;
};

// keys [lo, hi) that row t of the sequence may see
struct Range {
    int lo, hi;
};
__device__ __forceinline__ Range visible(const AttnArgs& a, const Seq& s, int t) {
    if (!a.causal) return {0, s.keys};
    const int i = s.len - s.n + t;
    // (max(0, i - window) without overflow, i may be negative)
    return {i - min(i, a.window), min(s.keys, i + 1)};
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
// r / G, head r % G of the group), cut into tiles; a tile has as many key steps (64 keys) as its rows see.  The lengths are
// known on the device only, so that is where the work of a key head is dealt out to its workgroups ("parts"), in one of three
// ways, whichever ends first by the counts of steps and what a piece of a tile costs:
//   kWhole  whole tiles, the last (longest) ones of the sequences first, in turns there and back over the parts;
//   kEven   every tile in equal pieces, one piece to a part: the shortest pieces that give no more of them than parts;
//   kLine   the steps of all tiles stand in one line and every part takes an equal stretch of it, wherever tiles begin and
//           end: perfect balance however unequal the lengths, at the price of two or more pieces in a part.
// (A prompt of 4096 tokens, 32 heads, on 8 parts a head: 190 us in whole tiles, 258 in a line.)
// A piece that is not a whole tile leaves an unnormalised result, which join_kernel puts together.  Every workgroup computes
// the same plan from the same numbers, and so does a recorded call that is replayed on new ones.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kKeyStep = 64;

struct Plan {
    int rows;       // rows of a tile (a power of two)
    int waves;      // of a workgroup (few-rows kernel)
    int lo, hi;     // sequences with lo <= n * G <= hi belong to this kernel
    int parts;      // workgroups per key head; 0: no pieces, the grid has a workgroup for every tile there may be
    int min_steps;  // fewest steps worth a workgroup
    int piece_cost, join_cost;  // of a piece of a tile, and of joining them, in steps
    int even;       // kEven is worth looking for
    int* joins;     // [parts][Hkv][kJoinInts]: the tile a part begins inside of, if it is the first part to do so
    float* o;       // partial results [2 * part + (not the part's first piece)][Hkv][rows][D], unnormalised
    float* ml;      // [..][rows][2]: maximum (base 2, scaled) and sum
};

// n_pieces (0: nothing to join) | first packed row of the sequence | first row of the tile | rows of the tile that exist |
// part the tile begins in | 1 if it is not that part's first piece
constexpr int kJoinInts = 8;

__device__ __forceinline__ int tiles_of(const AttnArgs& a, const Plan& p, const Seq& q) {
    const int64_t rows = (int64_t)q.n * a.G;
    return rows < 1 || rows < p.lo || rows > p.hi ? 0 : (int)((rows + p.rows - 1) >> (31 - __builtin_clz(p.rows)));
}
// key steps [first, first + steps) of tile t; a tile that sees nothing has one (its result is still stored)
__device__ __forceinline__ void steps_of(const AttnArgs& a, const Plan& p, const Seq& q, int t, int& first, int& steps) {
    const int last_row = (int)min((int64_t)(t + 1) * p.rows, (int64_t)q.n * a.G) - 1;
    first = visible(a, q, t * p.rows / a.G).lo / kKeyStep;
    steps = max(1, (visible(a, q, last_row / a.G).hi + kKeyStep - 1) / kKeyStep - first);
}

__device__ __forceinline__ int64_t lane64(int64_t x, int from) {  // (from: the same in every lane)
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, from);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), from);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}
// A value of another lane of the same row of 16, or of the row(s) before, by data-parallel primitives (one instruction where a
// shuffle through LDS takes a hundred clocks; these stand at the start of every call).  Lanes without a source get `none`.
template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ int dpp(int x, int none) {
    return __builtin_amdgcn_update_dpp(none, x, kCtrl, kRowMask, 0xf, false);
}
// running combination over the lanes: shifts by 1, 2, 4, 8 inside rows of 16, then the last lanes of rows 0 / 2 and of row 1
template <typename F>
__device__ __forceinline__ int scan_lanes(int x, int none, F f) {
    x = f(x, dpp<0x111>(x, none));
    x = f(x, dpp<0x112>(x, none));
    x = f(x, dpp<0x114>(x, none));
    x = f(x, dpp<0x118>(x, none));
    x = f(x, dpp<0x142, 0xa>(x, none));
    return f(x, dpp<0x143, 0xc>(x, none));
}
__device__ __forceinline__ int scan32(int x) {  // sum over the lanes up to this one
    return scan_lanes(x, 0, [](int a, int b) { return a + b; });
}
template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ int64_t dpp64(int64_t x) {
    const uint32_t lo = (uint32_t)dpp<kCtrl, kRowMask>((int)(uint32_t)x, 0), hi = (uint32_t)dpp<kCtrl, kRowMask>((int)(x >> 32), 0);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t scan64(int64_t x) {
    x += dpp64<0x111>(x);
    x += dpp64<0x112>(x);
    x += dpp64<0x114>(x);
    x += dpp64<0x118>(x);
    x += dpp64<0x142, 0xa>(x);
    return x + dpp64<0x143, 0xc>(x);
}
__device__ __forceinline__ int wave_most(int x) {
    return __builtin_amdgcn_readlane(scan_lanes(x, (int)0x80000000, [](int a, int b) { return max(a, b); }), 63);
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(scan32(x), 63); }
// x * i / n, rounded down (x * i below 2^62)
__device__ __forceinline__ int64_t mul_div(int64_t x, int i, int n) {
    if (x < (1 << 22) && i <= 512) return (int64_t)((uint32_t)x * (uint32_t)i / (uint32_t)n);
    return x * i / n;
}

// kWhole: which tile, counted from the last, is the j-th of part i -- there and back, so that the lengths even out
__device__ __forceinline__ int whole_turn(int j, int i, int parts) { return j * parts + (j & 1 ? parts - 1 - i : i); }

struct Piece {
    int s, tile;       // sequence, row tile
    Seq q;
    int first, steps;  // key steps of the whole tile
    int from;          // of them (kLine), or of its pieces (kEven), where the position lies
};

enum Deal : int { kWhole, kEven, kLine };

// The line of one key head's tiles, held by a wave: 64 tiles at a time, one in each lane.
struct Line {
    int base;             // number of lane 0's tile
    int s, t;             // of this lane's tile: sequence, tile of the sequence
    Seq q;
    int first, steps;     // its key steps (steps 0: there is no such tile)
    int64_t before, sum;  // weights before this block of tiles; in it, up to and with this lane's
    int64_t total;        // of the whole line
    int n_tiles;
    int parts;            // workgroups that share the line (at most p.parts)
    int deal;             // weight of a tile: 1, its pieces, its steps
    int per;              // kEven: longest piece

    // Tiles base .. base + 63: each lane looks for its tile in the running count of tiles over the sequences.  A sequence's
    // rows begin where all before it have ended, whatever cu says: no row belongs to two, so there are no more tiles than rows.
    __device__ __forceinline__ void block(const AttnArgs& a, const Plan& p, int base_, int lane) {
        base = base_;
        steps = 0, first = 0, s = 0, t = 0, q = Seq{0, 0, 0, 0};
        int seen = 0, ended = 0;
        for (int sb = 0; sb < a.g.S; sb += kWave) {
            Seq x = {0, 0, 0, 0};
            if (sb + lane < a.g.S) x = seq_of(a.g, sb + lane);
            const int from = max(scan_lanes(x.q0, 0, [](int a, int b) { return max(a, b); }), ended);
            x.n = max(x.q0 + x.n - from, 0);
            x.q0 = from;
            ended = __builtin_amdgcn_readlane(from, 63);
            const int mine = tiles_of(a, p, x);
            const int upto = scan32(mine);
            const int here = __builtin_amdgcn_readlane(upto, 63);
            const int want = base + lane - seen;
            if (base + kWave > seen && base < seen + here) {  // (uniform: some lane's tile is one of these sequences')
                int at = 0;
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) at += __shfl(upto, at + o - 1, 64) <= want ? o : 0;
                const int start = __shfl(upto - mine, at, 64);
                const Seq y = {__shfl(x.q0, at, 64), __shfl(x.n, at, 64), __shfl(x.len, at, 64), __shfl(x.keys, at, 64)};
                if (want >= 0 && want < here) {
                    s = sb + at, t = want - start, q = y;
                    steps_of(a, p, q, t, first, steps);
                }
            }
            seen += here;
        }
        n_tiles = seen;
        weigh();
    }
    __device__ __forceinline__ void weigh() {
        sum = scan64(deal == kLine ? steps : steps == 0 ? 0 : deal == kEven ? (steps + per - 1) / per : 1);
    }
    __device__ __forceinline__ void init(const AttnArgs& a, const Plan& p, int lane) {
        deal = p.parts ? kLine : kWhole;
        per = 1;
        block(a, p, 0, lane);
        before = 0;
        total = lane64(sum, 63);
        parts = 0;
        if (p.parts) {
            int longest = wave_most(steps);
            if (n_tiles > kWave) {
                for (int b = kWave; b < n_tiles; b += kWave) {
                    block(a, p, b, lane);
                    total += lane64(sum, 63);
                    longest = max(longest, wave_most(steps));
                }
                block(a, p, 0, lane);
            }
            parts = total >= (int64_t)p.parts * p.min_steps ? p.parts : max(1, (int)total / p.min_steps);
            // whole tiles: the most that a part gets; beyond a wave of tiles, as if all were as long as the longest
            const int rounds = (n_tiles + p.parts - 1) / p.parts;
            int64_t whole = (int64_t)longest * rounds;
            if (n_tiles <= kWave && rounds > 1) {
                int load = 0;
                for (int j = 0; j < rounds; ++j) {
                    const int at = n_tiles - 1 - whole_turn(j, lane, p.parts);
                    const int x = __shfl(steps, max(at, 0), 64);
                    load += lane < p.parts && at >= 0 ? x : 0;
                }
                whole = wave_most(load);
            }
            whole += (rounds - 1) * p.piece_cost;
            const int64_t fair = mul_div(total, 1, parts);
            int64_t best = fair + (n_tiles > 1 ? 1 + rounds : 1) * p.piece_cost + p.join_cost;
            if (whole <= best) deal = kWhole, best = whole;
            if (p.even && n_tiles > 1 && n_tiles <= min(parts, kWave)) {
                int lo = (int)fair, hi = longest;  // lo pieces: too many, hi: few enough
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if (wave_total((steps + mid - 1) / mid) <= parts) hi = mid;
                    else lo = mid;
                }
                if (hi < longest && hi + p.piece_cost + p.join_cost < best) deal = kEven, per = hi;
            }
            if (deal != kLine) {
                weigh();
                total = lane64(sum, 63);  // (kEven: one block of tiles)
            }
        }
        if (deal == kWhole) total = n_tiles;
    }
    __device__ __forceinline__ int64_t start(int i) const { return mul_div(total, i, parts); }  // kLine: of part i
    __device__ __forceinline__ int part_of(int64_t x) const {
        if (total < (1 << 22) && parts <= 512) return (int)((uint32_t)((x + 1) * parts - 1) / (uint32_t)total);
        return (int)(((x + 1) * parts - 1) / total);
    }

    // the tile at position x < total; positions of later calls do not decrease.  (steps = 0: there is none -- the lengths have
    // changed under the call, which has to end all the same)
    __device__ __forceinline__ Piece find(const AttnArgs& a, const Plan& p, int64_t x, int lane) {
        while (x >= before + lane64(sum, 63) && base + kWave < n_tiles) {
            before += lane64(sum, 63);
            block(a, p, base + kWave, lane);
        }
        const uint64_t vote = __builtin_amdgcn_ballot_w64(x < before + sum);
        Piece r;
        r.steps = 0;
        if (vote == 0) return r;
        const int at = __builtin_ctzll(vote);
        r.s = __builtin_amdgcn_readlane(s, at);
        r.tile = __builtin_amdgcn_readlane(t, at);
        r.q = Seq{__builtin_amdgcn_readlane(q.q0, at), __builtin_amdgcn_readlane(q.n, at),
                  __builtin_amdgcn_readlane(q.len, at), __builtin_amdgcn_readlane(q.keys, at)};
        r.first = __builtin_amdgcn_readlane(first, at);
        r.steps = __builtin_amdgcn_readlane(steps, at);
        r.from = (int)(x - before - (at ? lane64(sum, at - 1) : 0));
        return r;
    }
};

// What a workgroup does: calls work(piece, first step, steps, whole, place in the workspace) for each of its pieces.  (The
// line's block is made again behind a piece, so that it takes no registers meanwhile.)
template <typename F>
__device__ __forceinline__ void for_each_piece(const AttnArgs& a, const Plan& p, int lane, F&& work) {
    const int me = (int)(blockIdx.x / (unsigned)a.Hkv), n_wgs = (int)(gridDim.x / (unsigned)a.Hkv);
    int* note = p.joins + blockIdx.x * kJoinInts;
    if (p.parts && threadIdx.x == 0) note[0] = 0;
    Line line;
    line.init(a, p, lane);
    const int deal = line.deal;
    int64_t x = 0, end = 0;
    int turn = 0;
    if (deal == kLine) {
        if (me < line.parts) x = line.start(me), end = line.start(me + 1);
    } else if (deal == kEven) {
        x = me, end = min(line.total, (int64_t)me + 1);
    } else {
        x = line.total - 1 - me;  // (downwards, the last and longest ones first)
    }
    if (deal == kWhole ? x < 0 : x >= end) return;
    const int64_t begin = x;
    for (;;) {
        if (deal == kWhole && (x < line.base || x >= line.base + kWave)) {
            line.before = x & ~(int64_t)(kWave - 1);
            line.block(a, p, (int)line.before, lane);
        }
        const Piece u = line.find(a, p, x, lane);
        if (u.steps == 0) return;
        int from = 0, n = u.steps, pieces = 1, i0 = me, shift = 0;
        if (deal == kLine) {
            from = u.from;
            n = (int)min((int64_t)(u.steps - from), end - x);
            const int64_t tile = x - from;
            i0 = line.part_of(tile);
            pieces = line.part_of(tile + u.steps - 1) - i0 + 1;
            shift = tile == line.start(i0) ? 0 : 1;
        } else if (deal == kEven) {
            pieces = (u.steps + line.per - 1) / line.per;
            from = (int)mul_div(u.steps, u.from, pieces);
            n = (int)mul_div(u.steps, u.from + 1, pieces) - from;
            i0 = me - u.from;
        }
        if (n < 1) return;
        if (pieces > 1 && x == begin && from > 0 && i0 == me - 1 && threadIdx.x == 0) {
            note[0] = pieces;
            note[1] = u.q.q0;
            note[2] = u.tile * p.rows;
            note[3] = min(p.rows, u.q.n * a.G - u.tile * p.rows);
            note[4] = i0;
            note[5] = shift;
        }
        work(u, u.first + from, n, pieces == 1, 2 * me + (x == begin ? 0 : 1));
        if (deal == kLine) x += n;
        else if (deal == kEven) x += 1;
        else x = line.total - 1 - whole_turn(++turn, me, n_wgs);
        if (deal == kWhole ? x < 0 : x >= end) return;
        line.block(a, p, line.base, lane);
    }
}

// Kernels that use more than 64 KB of LDS need the limit raised once per device: `dev`, the one that owns the operands.
template <auto kKernel>
int raise_lds(int dev, int bytes) {
    static std::mutex mutex;
    static std::atomic<bool> raised[kMaxDevices];
    if (raised[dev].load(std::memory_order_acquire)) return VQA_OK;
    std::lock_guard<std::mutex> lock(mutex);
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        hipSuccess) {
        (void)hipGetLastError();
        return VQA_ERR_LAUNCH_FAILED;
    }
    raised[dev].store(true, std::memory_order_release);
    return VQA_OK;
}

template <typename Tag>
int launch_few(const AttnArgs& a, const Plan& p, int D, bool e4m3, int64_t grid, int dev, hipStream_t stream);
template <typename Tag>
int launch_chunk(const AttnArgs& a, const Plan& p, int D, bool e4m3, int64_t grid, int dev, hipStream_t stream);

}  // namespace paged
}  // namespace vqa
