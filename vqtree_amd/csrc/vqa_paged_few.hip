// Few rows, many keys: generation steps, drafted tokens, short chunks (vqa_paged_attn_*).  HBM bound: every key and value
// row of a (sequence, key head) is read once for all rows of a tile, 16 * NB of them (grouped query heads and new tokens
// together).  Measured (kernel time): 16 sequences, 260 000 keys together, 32 query and 8 key heads, head dim 128: 185 us for
// 1.19 GB of 16-bit rows, 6.4 TB/s (reads alone reach about 7); 65 536 keys of 32 heads in e4m3: 92 us for 0.54 GB, 5.9 TB/s.
// One sequence of 1000 keys is latency: 13 us -- 2 until the work is dealt out, 1 until the first tile is asked for, 4 for
// four tiles per wave, 3 to join the waves.
//
// One workgroup of 8 waves, or 4 where there are enough tiles for two workgroups on a compute unit (the start and the end of
// one under the loads of the other), works on one piece of a tile's keys at a time; its waves take consecutive parts of it and
// never wait for each other until their results are joined at the end.  A wave walks 32-key tiles: the rows go HBM -> LDS directly
// (global_load_lds_dwordx4, whole rows per instruction, no registers), S^T = K.Q^T and O^T = V^T.P^T run on
// v_mfma_f32_16x16x32 -- the matrix pipe has room to spare at any memory rate, so a single query row goes through it too.
//
// Layouts.  MFMA row 4 * quad + r of key block kb stands for key 8 * quad + 4 * kb + r of the tile, so the lane (n = row,
// quad) holds the scores of keys 8 * quad .. + 7 of its row: the B operand of the P.V product as it is.  Its V^T operand is
// read by transposing LDS reads: ds_read_b64_tr_b16 (4 keys of one d per lane, twice) or, from e4m3 rows,
// ds_read_b64_tr_b8 (8 keys).  Tiles are stored with the 16-byte (K) or 32-byte (V) pieces of a row XORed by a function of
// the row, such that the rows one read touches lie in different banks.
//
// e4m3: keys are widened to the element type by v_cvt_scalef32_pk_* with their row's factor (a lane reads one key); values
// are widened without factor, always to bf16 (exact), and the factor of the key goes to the probability instead, since a lane
// then holds 8 keys of one d.
//
// Where the P.V product is in bf16, a probability is split into two bf16 numbers (16 bits together): the matrix pipe has the
// time, and the output's error against 64 bits falls from 1.4 times that of its own rounding to 1.0 times.  In f16 (16-bit
// pages) a probability has 11 bits as it is, and the error is 1.1 to 1.4 times that of the rounding.
#include "vqa_flash2.h"
#include "vqa_paged_attn.h"

namespace vqa {
namespace paged {
namespace few {

using flash::u32x4_t;
typedef flash::s16x4_t s16x4_t;
typedef int i32x2_t __attribute__((ext_vector_type(2)));

constexpr int kKeys = 32;    // keys per tile
constexpr float kLazy = 8.f; // a row's reference maximum moves when a tile exceeds it by 2^kLazy

template <int D, bool kE4m3>
struct Geo {
    static constexpr int kRow = kE4m3 ? D : 2 * D;       // bytes of a stored row
    static constexpr int kChunks = kRow / 16;            // 16-byte pieces per row: 4, 8 or 16
    static constexpr int kRowsPerLoad = 64 / kChunks;    // rows one direct-to-LDS load brings
    static constexpr int kLoads = kKeys / kRowsPerLoad;  // loads per tile and source
    static constexpr int kTile = kKeys * kRow;
    static constexpr int kRing = 8192 / kTile;           // tiles of each source in flight per wave
    static constexpr int kExp = kE4m3 ? 64 : 0;          // exponents: 32 of the keys, 32 of the values
    static constexpr int kSlot = 2 * kTile + kExp;       // keys | values | exponents
    static constexpr int kWaveBytes = kRing * kSlot;
    static constexpr int kSteps = D / 32;                // k-steps of the score product
    static constexpr int kDBlocks = D / 16;
    static constexpr int kKLoads = kLoads + (kE4m3 ? 1 : 0);

    // XOR of the 16-byte piece index of key row r: 16 lanes read the same piece of rows {0-3, 8-11, 16-19, 24-27} (+ 4)
    static __device__ __forceinline__ int swz_k(int r) {
        if constexpr (kChunks == 16) return (r & 3) | (((r >> 3) & 3) << 2);
        if constexpr (kChunks == 8) return ((r >> 1) & 1) | (((r >> 3) & 3) << 1);
        return (r >> 3) & 3;
    }
    // of value row r.  16 bits: 32 lanes read the same 32-byte piece of rows {0-3, 8-11} (+ 4, + 16); e4m3: the same 16-byte
    // piece of 16 consecutive rows
    static __device__ __forceinline__ int swz_v(int r) {
        if constexpr (kE4m3) return kChunks == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
        if constexpr (kChunks == 16) return 2 * ((r & 3) | (((r >> 3) & 1) << 2));
        return 2 * (((r >> 1) & 1) | (((r >> 3) & 1) << 1));
    }
};

template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// joins the four lanes (quads) that hold one row
__device__ __forceinline__ float quads_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float quads_sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}

// Brings tiles of one wave.  kOnce: no other tile reads these rows (all rows of a sequence fit one tile), so the loads are
// marked non-temporal: 213 -> 189 us for 1.19 GB of 16-bit rows, 105 -> 95 us for 0.54 GB of e4m3 rows.
template <int D, bool kE4m3>
struct Loader {
    typedef Geo<D, kE4m3> G;
    const char *k, *v;             // pools at the key head
    const uint8_t *ke, *ve;
    const int32_t* table;          // of the sequence
    int end;                       // keys from here on are not there
    int lane;
    int tab, tab0;                 // table entries tab0 + lane
    uint32_t lds;                  // of the wave
    uint32_t k_off[G::kLoads], v_off[G::kLoads];  // this lane's byte in a whole group of rows, per load

    static __device__ __forceinline__ int row_of_load(int i, int lane) { return (i * G::kRowsPerLoad) % 16 + lane / G::kChunks; }
    template <bool kV>
    static __device__ __forceinline__ uint32_t piece_of(int i, int lane) {
        const int full = i * G::kRowsPerLoad + lane / G::kChunks;
        return (uint32_t)((lane % G::kChunks) ^ (kV ? G::swz_v(full) : G::swz_k(full))) * 16u;
    }
    __device__ __forceinline__ void init(const AttnArgs& a, int h, uint32_t lds_, int lane_) {
        k = a.kp.p + h * a.kp.sh, v = a.vp.p + h * a.vp.sh;
        if constexpr (kE4m3) ke = a.kp.e + h * a.kp.eh, ve = a.vp.e + h * a.vp.eh;
        lds = lds_, lane = lane_;
#pragma unroll
        for (int i = 0; i < G::kLoads; ++i) {
            k_off[i] = (uint32_t)row_of_load(i, lane) * (uint32_t)a.kp.sn + piece_of<false>(i, lane);
            v_off[i] = (uint32_t)row_of_load(i, lane) * (uint32_t)a.vp.sn + piece_of<true>(i, lane);
        }
    }
    __device__ __forceinline__ void sequence(const AttnArgs& a, int s, int end_) {
        table = a.g.table + (int64_t)s * a.g.table_ss;
        end = end_;
        tab0 = -0x40000000;
        tab = -1;
    }
    // page of key j (below the table's end), -1 if it is not there
    __device__ __forceinline__ int page_at(const Seqs& g, int j) {
        const int c = j >> g.page_shift;
        if (c - tab0 >= 64 || c < tab0) {  // (uniform)
            tab0 = c;
            tab = c + lane < g.width ? table[c + lane] : -1;
            if ((unsigned)tab >= (unsigned)g.n_pages) tab = -1;
        }
        return __builtin_amdgcn_readlane(tab, c - tab0);
    }
    // Where the two 16-row groups of tile [j0, j0 + 32) lie.  Rows from `end` on repeat the last one that is there; a page
    // that is not there reads page 0 (its keys are hidden).
    struct Place {
        int page[2], j[2];
        int there;  // a bit per group
    };
    __device__ __forceinline__ Place place(const Seqs& g, int j0) {
        Place x;
        x.there = 0;
#pragma unroll
        for (int gi = 0; gi < 2; ++gi) {
            x.j[gi] = j0 + 16 * gi < end ? j0 + 16 * gi : (end - 1) & ~15;
            const int p = page_at(g, x.j[gi]);
            x.there |= p >= 0 ? 1 << gi : 0;
            x.page[gi] = max(p, 0);
        }
        return x;
    }
    template <bool kV, bool kOnce>
    __device__ __forceinline__ void request(const AttnArgs& a, const Place& x, int slot) {
        const uint32_t dst = lds + (uint32_t)(slot * G::kSlot) + (kV ? G::kTile : 0);
        const Pool& pool = kV ? a.vp : a.kp;
        const int in_page = (1 << a.g.page_shift) - 1;
        const char* group[2];
#pragma unroll
        for (int gi = 0; gi < 2; ++gi)
            group[gi] = (kV ? v : k) + (int64_t)x.page[gi] * pool.sp + (int64_t)(x.j[gi] & in_page) * pool.sn;
        if (x.j[1] + 16 <= end && x.j[0] != x.j[1]) {
            flash2::static_for<G::kLoads>([&](auto I) {
                constexpr int i = decltype(I)::value;
                issue<i, kOnce>(dst, kV ? v_off[i] : k_off[i], group[i * G::kRowsPerLoad / 16]);
            });
        } else {
            flash2::static_for<G::kLoads>([&](auto I) {
                constexpr int i = decltype(I)::value;
                constexpr int gi = i * G::kRowsPerLoad / 16;
                const uint32_t row = (uint32_t)min(row_of_load(i, lane), end - 1 - x.j[gi]);
                issue<i, kOnce>(dst, row * (uint32_t)pool.sn + piece_of<kV>(i, lane), group[gi]);
            });
        }
        if constexpr (kE4m3 && !kV) {
            // lanes 0, 1: exponents of the two groups' keys, 2, 3: of their values
            if (lane < 4) {
                const int64_t page = lane & 1 ? x.page[1] : x.page[0];
                const int at = (lane & 1 ? x.j[1] : x.j[0]) & in_page;
                flash::dma16((lane < 2 ? ke + page * a.kp.ep : ve + page * a.vp.ep) + at,
                             lds + (uint32_t)(slot * G::kSlot + 2 * G::kTile));
            }
        }
    }
    template <int I, bool kOnce>
    static __device__ __forceinline__ void issue(uint32_t dst, uint32_t off, const char* base) {
        // (a load may not follow the write of M0 directly)
        if constexpr (kOnce)
            asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3 nt"
                         :
                         : "s"(dst), "n"(I * 1024), "v"(off), "s"(base)
                         : "memory", "scc");
        else
            asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3"
                         :
                         : "s"(dst), "n"(I * 1024), "v"(off), "s"(base)
                         : "memory", "scc");
    }
};

// kBlocks: rows of a tile in blocks of 16.  In tiles of two a sequence that has one is done as one, so single tokens do not pay
// for the drafts and short chunks they share a call with (generation step of 16 sequences: two blocks 223 us, one 193).
template <typename Tag, int D, bool kE4m3, int kBlocks, int kWaves>
__global__ __launch_bounds__(kWaves * 64, 2) void few_kernel(AttnArgs a, Plan p) {
    typedef Geo<D, kE4m3> G;
    typedef typename Elem<Tag>::vec8 vec8;
    typedef typename std::conditional<kE4m3, bf16_tag, Tag>::type PTag;  // element type of the P.V product
    typedef typename Elem<PTag>::vec8 pvec8;
    constexpr bool kSplitP = std::is_same<PTag, bf16_tag>::value;
    constexpr int kTileRows = 16 * kBlocks;
    constexpr int kStageRow = D + 4;  // floats; the padding spreads a column of rows over the banks
    typedef const __attribute__((address_space(3))) u32x4_t* lds16_ptr;
    typedef __attribute__((address_space(3))) s16x4_t* lds_tr_ptr;
    typedef __attribute__((address_space(3))) i32x2_t* lds_tr8_ptr;
    typedef const __attribute__((address_space(3))) uint8_t* lds_u8_ptr;
    typedef const __attribute__((address_space(3))) i32x2_t* lds8_ptr;
    extern __shared__ __attribute__((aligned(1024))) char smem[];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, quad = lane >> 4;
    const int h = __builtin_amdgcn_readfirstlane((int)(blockIdx.x % (unsigned)a.Hkv));
    const uint32_t lds0 = flash::lds_addr_of(smem);
    Loader<D, kE4m3> ld;
    ld.init(a, h, lds0 + (uint32_t)(wave * G::kWaveBytes), lane);

    auto piece = [&](auto blocks, const Piece& u, int step, int n_steps, bool whole, int slot_out) __attribute__((always_inline)) {
        constexpr int NB = decltype(blocks)::value, kRows = 16 * NB;
        constexpr bool kOnce = NB == 1;
        const Seq& q = u.q;
        const int row0 = u.tile * kTileRows;
        const int n_rows = min(kRows, q.n * a.G - row0);  // (a tile is of one sequence: fits 32 bits)
        const int u_lo = step * kKeyStep;
        const int u_hi = (int)min((int64_t)(step + n_steps) * kKeyStep, (int64_t)q.keys);
        // this wave's part, in tiles
        const int n_tiles = max(0, (u_hi - u_lo + kKeys - 1) / kKeys);
        const int t_lo = n_tiles * wave / kWaves, t_hi = n_tiles * (wave + 1) / kWaves;

        ld.sequence(a, u.s, u_hi);
        typename Loader<D, kE4m3>::Place places[G::kRing];
        auto ask_k = [&](int t, int slot) __attribute__((always_inline)) {
            places[slot] = ld.place(a.g, u_lo + t * kKeys);
            ld.template request<false, kOnce>(a, places[slot], slot);
        };
        auto ask_v = [&](int slot) __attribute__((always_inline)) { ld.template request<true, kOnce>(a, places[slot], slot); };
#pragma unroll
        for (int i = 0; i < G::kRing; ++i)
            if (t_lo + i < t_hi) ask_k(t_lo + i, i), ask_v(i);

        // rows of this lane's columns: what they see, and their queries (rows past the end repeat the last)
        int lo[NB], hi[NB];
        vec8 qf[NB][G::kSteps];
        int all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int r = row0 + min(b * 16 + n, n_rows - 1);
            const int t = r / a.G, g = r - t * a.G;
            const Range v = visible(a, q, t);
            lo[b] = v.lo, hi[b] = v.hi;
            const uint16_t* src = a.q + (int64_t)(q.q0 + t) * a.q_st + (int64_t)(h * a.G + g) * a.q_sh;
#pragma unroll
            for (int k = 0; k < G::kSteps; ++k) {
                const int d = kE4m3 ? ((k / 2) * 4 + quad) * 16 + (k % 2) * 8 : k * 32 + quad * 8;
                qf[b][k] = *reinterpret_cast<const vec8*>(src + d);
            }
        }
        {   // what every row of the tile sees: the first row's end and the last row's start
            const int t0 = row0 / a.G, t1 = (row0 + n_rows - 1) / a.G;
            all_hi = visible(a, q, t0).hi, all_lo = visible(a, q, t1).lo;
        }

        float m[NB], l[NB];
        f32x4_t o[NB][G::kDBlocks];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            m[b] = -INFINITY, l[b] = 0.f;
#pragma unroll
            for (int d = 0; d < G::kDBlocks; ++d) o[b][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }

        // per-lane LDS addresses inside a slot
        const int k_row[2] = {(n >> 2) * 8 + (n & 3), (n >> 2) * 8 + 4 + (n & 3)};  // key of this lane's MFMA row, per block
        auto tile = [&](int t, int slot) __attribute__((always_inline)) {
            const int j0 = u_lo + t * kKeys;
            const uint32_t base = ld.lds + (uint32_t)(slot * G::kSlot);
            const bool full = t + G::kRing < t_hi;  // the ring is refilled behind this tile
            if (t + G::kRing - 1 < t_hi)
                wait_loads<G::kRing * G::kLoads + (G::kRing - 1) * G::kKLoads>();
            else
                wait_loads<0>();
            f32x4_t s[NB][2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int row = k_row[kb];
                const uint32_t row_addr = base + (uint32_t)(row * G::kRow);
                vec8 kf[G::kSteps];
                if constexpr (kE4m3) {
                    const float f = factor_of(*(lds_u8_ptr)(uintptr_t)(base + 2 * G::kTile + row));
#pragma unroll
                    for (int c = 0; c < G::kSteps / 2; ++c) {
                        const u32x4_t w = *(lds16_ptr)(uintptr_t)(row_addr + (uint32_t)(((c * 4 + quad) ^ G::swz_k(row)) * 16));
                        const uint2 w0 = widen4<Tag>(w[0], f), w1 = widen4<Tag>(w[1], f);
                        const uint2 w2 = widen4<Tag>(w[2], f), w3 = widen4<Tag>(w[3], f);
                        kf[2 * c] = __builtin_bit_cast(vec8, u32x4_t{w0.x, w0.y, w1.x, w1.y});
                        kf[2 * c + 1] = __builtin_bit_cast(vec8, u32x4_t{w2.x, w2.y, w3.x, w3.y});
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < G::kSteps; ++k)
                        kf[k] = __builtin_bit_cast(
                            vec8, *(lds16_ptr)(uintptr_t)(row_addr + (uint32_t)(((k * 4 + quad) ^ G::swz_k(row)) * 16)));
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < G::kSteps; ++k) acc = Elem<Tag>::mfma16(kf[k], qf[b][k], acc);
                    s[b][kb] = acc;
                }
            }
            uint32_t vexp[2] = {0, 0};
            if constexpr (kE4m3) {
                const i32x2_t e = *(lds8_ptr)(uintptr_t)(base + 2 * G::kTile + 32 + quad * 8);
                vexp[0] = (uint32_t)e[0], vexp[1] = (uint32_t)e[1];
            }
            const int there = places[slot].there;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile's keys are in registers: the slot may be refilled
            if (full) ask_k(t + G::kRing, slot);

            const bool plain = j0 >= all_lo && j0 + kKeys <= all_hi && there == 3;  // (uniform)
            if (!plain) {
                const bool mine = (there >> (quad >> 1)) & 1;  // keys 8 * quad .. + 7 lie in one group of 16
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int j = j0 + quad * 8 + e;
                        const bool seen = mine && j >= lo[b] && j < hi[b];
                        s[b][e >> 2][e & 3] = seen ? s[b][e >> 2][e & 3] : -INFINITY;
                    }
            }
            pvec8 pf[NB], pl[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float mx = s[b][0][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[b][e >> 2][e & 3]);
                mx *= a.scale_log2e;
                if (__builtin_amdgcn_ballot_w64(mx > (m[b] == -INFINITY ? -INFINITY : m[b] + kLazy))) {
                    mx = quads_max(mx);
                    const bool up = mx > (m[b] == -INFINITY ? -INFINITY : m[b] + kLazy);
                    const float alpha = up ? fast_exp2(m[b] - mx) : 1.f;
                    m[b] = up ? mx : m[b];
                    l[b] *= alpha;
#pragma unroll
                    for (int d = 0; d < G::kDBlocks; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[b][d][e] *= alpha;
                }
                const float ref = m[b] == -INFINITY ? 0.f : m[b];
                float pr[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    pr[e] = fast_exp2(__builtin_fmaf(s[b][e >> 2][e & 3], a.scale_log2e, -ref));
                    l[b] += pr[e];
                    if constexpr (kE4m3)
                        pr[e] = __builtin_ldexpf(pr[e], max((int)((vexp[e >> 2] >> (8 * (e & 3))) & 0xffu), 1) - 127);
                }
                const u32x4_t pk = {Elem<PTag>::pack2(pr[0], pr[1]), Elem<PTag>::pack2(pr[2], pr[3]),
                                    Elem<PTag>::pack2(pr[4], pr[5]), Elem<PTag>::pack2(pr[6], pr[7])};
                pf[b] = __builtin_bit_cast(pvec8, pk);
                if constexpr (kSplitP) {
                    u32x4_t rest;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        rest[e] = Elem<PTag>::pack2(pr[2 * e] - Elem<PTag>::from_bits((uint16_t)(pk[e] & 0xffffu)),
                                                    pr[2 * e + 1] - Elem<PTag>::from_bits((uint16_t)(pk[e] >> 16)));
                    pl[b] = __builtin_bit_cast(pvec8, rest);
                }
            }

            if (full)
                wait_loads<G::kRing * G::kKLoads + (G::kRing - 1) * G::kLoads>();
            else
                wait_loads<0>();
#pragma unroll
            for (int d = 0; d < G::kDBlocks; ++d) {
                pvec8 vf;
                if constexpr (kE4m3) {
                    const int row = quad * 8 + (n >> 1);
                    const uint32_t addr = base + G::kTile + (uint32_t)(row * G::kRow + ((d ^ G::swz_v(row)) * 16) + (n & 1) * 8);
                    const i32x2_t w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_tr8_ptr)(uintptr_t)addr);
                    const uint2 w0 = widen4<PTag>((uint32_t)w[0], 1.f), w1 = widen4<PTag>((uint32_t)w[1], 1.f);
                    vf = __builtin_bit_cast(pvec8, u32x4_t{w0.x, w0.y, w1.x, w1.y});
                } else {
                    const int row = quad * 8 + (n >> 2);
                    const uint32_t in_row = (uint32_t)(((2 * d + ((n & 3) >> 1)) * 16) + (n & 1) * 8);
                    const uint32_t a0 = base + G::kTile + (uint32_t)(row * G::kRow) + (in_row ^ (uint32_t)(G::swz_v(row) * 16));
                    const uint32_t a1 =
                        base + G::kTile + (uint32_t)((row + 4) * G::kRow) + (in_row ^ (uint32_t)(G::swz_v(row + 4) * 16));
                    const s16x4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(uintptr_t)a0);
                    const s16x4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(uintptr_t)a1);
                    const short __attribute__((ext_vector_type(8))) w = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
                    vf = __builtin_bit_cast(pvec8, w);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    o[b][d] = Elem<PTag>::mfma16(vf, pf[b], o[b][d]);
                    if constexpr (kSplitP) o[b][d] = Elem<PTag>::mfma16(vf, pl[b], o[b][d]);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (full) ask_v(slot);
        };
        for (int t = t_lo; t < t_hi; t += G::kRing) {
#pragma unroll
            for (int i = 0; i < G::kRing; ++i)
                if (t + i < t_hi) tile(t + i, i);
        }

        // join the waves: maxima and sums first, then the rows scaled to the common maximum, through LDS
        float* stage = reinterpret_cast<float*>(smem);                       // [wave][row][kStageRow]
        float* ml = stage + kWaves * kRows * kStageRow;                      // [wave][row][2]
        uint32_t* bad = reinterpret_cast<uint32_t*>(ml + kWaves * kRows * 2);
        __syncthreads();  // every wave is done with its tiles
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float lt = quads_sum(l[b]);
            if (quad == 0) {
                ml[(wave * kRows + b * 16 + n) * 2] = m[b];
                ml[(wave * kRows + b * 16 + n) * 2 + 1] = lt;
            }
        }
        if (threadIdx.x == 0) *bad = 0;
        __syncthreads();
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[(w * kRows + b * 16 + n) * 2]);
            const float f = m[b] == -INFINITY ? 0.f : fast_exp2(m[b] - top);
            float* row = stage + (wave * kRows + b * 16 + n) * kStageRow;
#pragma unroll
            for (int d = 0; d < G::kDBlocks; ++d)
                *reinterpret_cast<float4*>(row + d * 16 + quad * 4) =
                    make_float4(o[b][d][0] * f, o[b][d][1] * f, o[b][d][2] * f, o[b][d][3] * f);
        }
        __syncthreads();
        constexpr int kLanes = D / 8;  // threads per row, 8 elements each
        const int64_t part = ((int64_t)slot_out * a.Hkv + h) * kTileRows;
#pragma unroll
        for (int i = 0; i < kRows * kLanes / (kWaves * 64) + (kRows * kLanes % (kWaves * 64) ? 1 : 0); ++i) {
            const int at = i * kWaves * 64 + (int)threadIdx.x;
            const int r = at / kLanes, c = at % kLanes;
            if (r >= n_rows) continue;
            float top = -INFINITY, sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[(w * kRows + r) * 2]);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float mw = ml[(w * kRows + r) * 2];
                sum += ml[(w * kRows + r) * 2 + 1] * (mw == -INFINITY ? 0.f : fast_exp2(mw - top));
                const float* src = stage + (w * kRows + r) * kStageRow + c * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += src[e];
            }
            float probe = sum;
#pragma unroll
            for (int e = 0; e < 8; ++e) probe += v[e] * 0.f;
            if (!(probe < INFINITY)) atomicOr(bad + r / 32, 1u << (r % 32));
            if (!whole) {
                float* dst = p.o + (part + r) * D + c * 8;
                reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
                if (c == 0) {
                    p.ml[(part + r) * 2] = top;
                    p.ml[(part + r) * 2 + 1] = sum;
                }
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const int rr = row0 + r, t = rr / a.G, hq = h * a.G + rr - t * a.G;
                const u32x4_t pk = {Elem<Tag>::pack2(v[0] * inv, v[1] * inv), Elem<Tag>::pack2(v[2] * inv, v[3] * inv),
                                    Elem<Tag>::pack2(v[4] * inv, v[5] * inv), Elem<Tag>::pack2(v[6] * inv, v[7] * inv)};
                *reinterpret_cast<u32x4_t*>(a.out + (int64_t)(q.q0 + t) * a.o_st + (int64_t)hq * a.o_sh + c * 8) = pk;
                if (a.lse != nullptr && c == 0)
                    a.lse[(int64_t)(q.q0 + t) * a.Hq + hq] = sum == 0.f ? -INFINITY : top + fast_log2(sum);
            }
        }
        __syncthreads();
        // A row that came out as infinity or NaN may have met one in a value it does not see (0 * inf): done again key by key.
        uint64_t todo = *bad;
        for (int r = 0; todo; ++r, todo >>= 1) {
            if (!(todo & 1) || r % kWaves != wave) continue;
            const int rr = row0 + r, t = rr / a.G, hq = h * a.G + rr - t * a.G;
            const Range v = visible(a, q, t);
            RowState<D> st;
            row_by_lanes<Tag, D, kE4m3>(a, u.s, h, a.q + (int64_t)(q.q0 + t) * a.q_st + (int64_t)hq * a.q_sh, max(u_lo, v.lo),
                                        min(u_hi, v.hi), st, lane);
            if (!whole) {
#pragma unroll
                for (int e = 0; e < D / 64; ++e) p.o[(part + r) * D + lane * (D / 64) + e] = st.o[e];
                if (lane == 0) {
                    p.ml[(part + r) * 2] = st.m;
                    p.ml[(part + r) * 2 + 1] = st.l;
                }
            } else {
                store_row<Tag, D>(a, st, q.q0 + t, hq, lane);
            }
        }
        __syncthreads();  // the staging area is free for the next piece's tiles
    };
    for_each_piece(a, p, lane,
                   [&](const Piece& u, int step, int n_steps, bool whole, int slot_out) __attribute__((always_inline)) {
        if (kBlocks == 1 || u.q.n * a.G <= 16)
            piece(std::integral_constant<int, 1>(), u, step, n_steps, whole, slot_out);
        else
            piece(std::integral_constant<int, kBlocks>(), u, step, n_steps, whole, slot_out);
    });
}

template <int D, bool kE4m3, int NB, int kWaves>
constexpr int lds_bytes() {
    const int tiles = kWaves * Geo<D, kE4m3>::kWaveBytes;
    const int join = kWaves * 16 * NB * (D + 4) * 4 + kWaves * 16 * NB * 8 + 16;
    return tiles > join ? tiles : join;
}

template <typename Tag, int D, bool kE4m3, int NB, int kWaves>
int launch(const AttnArgs& a, const Plan& p, int64_t grid, int dev, hipStream_t stream) {
    constexpr int bytes = lds_bytes<D, kE4m3, NB, kWaves>();
    if (bytes > 64 * 1024) {
        if (int rc = raise_lds<few_kernel<Tag, D, kE4m3, NB, kWaves>>(dev, bytes)) return rc;
    }
    few_kernel<Tag, D, kE4m3, NB, kWaves><<<dim3((unsigned)grid), kWaves * 64, bytes, stream>>>(a, p);
    return launch_status();
}

template <typename Tag, int D, bool kE4m3>
int launch(const AttnArgs& a, const Plan& p, int64_t grid, int dev, hipStream_t stream) {
    if (p.waves == 4)
        return p.rows == 32 ? launch<Tag, D, kE4m3, 2, 4>(a, p, grid, dev, stream) : launch<Tag, D, kE4m3, 1, 4>(a, p, grid, dev, stream);
    return p.rows == 32 ? launch<Tag, D, kE4m3, 2, 8>(a, p, grid, dev, stream) : launch<Tag, D, kE4m3, 1, 8>(a, p, grid, dev, stream);
}

}  // namespace few

template <typename Tag>
int launch_few(const AttnArgs& a, const Plan& p, int D, bool e4m3, int64_t grid, int dev, hipStream_t stream) {
    if (D == 128)
        return e4m3 ? few::launch<Tag, 128, true>(a, p, grid, dev, stream) : few::launch<Tag, 128, false>(a, p, grid, dev, stream);
    return e4m3 ? few::launch<Tag, 64, true>(a, p, grid, dev, stream) : few::launch<Tag, 64, false>(a, p, grid, dev, stream);
}
template int launch_few<bf16_tag>(const AttnArgs&, const Plan&, int, bool, int64_t, int, hipStream_t);
template int launch_few<f16_tag>(const AttnArgs&, const Plan&, int, bool, int64_t, int, hipStream_t);

}  // namespace paged
}  // namespace vqa
