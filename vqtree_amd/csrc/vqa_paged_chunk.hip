// Many rows: chunks of prompts (vqa_paged_attn_*), on the software-pipelined core of vqa_flash2.h.  Bound by the issue of the
// core's instructions beside its matrix products.  Measured, 2048 new tokens behind 8192, 32 query and 8 key heads, head dim
// 128, 16 bits: 281 - 293 us a call among others, 1.06 - 1.10 PFLOP/s (a large library product: 1.35), matrix pipe 52 % busy;
// over an e4m3 cache 17 % more.  A workgroup takes 10 us until its first products and 7 to store its rows, 1.7 us per 64 keys
// between (e4m3: 12, 12 and 2.1), so short pieces pay for their ends.
//
// One workgroup of 4 waves owns a tile of 256 rows (grouped query heads and tokens together, so a chunk of 64 tokens with
// 4 query heads per key head fills one) and walks 64-key tiles of the piece it was given; a wave brings 16 rows of each
// tile, which lie in one page, so paging costs the key loop one look-up and two row addresses per tile, in scalar registers.
// Rows of a tile differ in what they see; masks are evaluated per element only on tiles where they do (diagonal, window
// edge, end, missing pages).
//
// e4m3 rows go HBM -> LDS as they are, each wave its own 16 of a tile, and are widened to the element type on the way into the
// tile buffers, once per workgroup: 8 conversions and two LDS writes per 1 KB and wave, dealt out over the score MFMAs (a
// wave converting the fragments it needs itself would do that work four times).  Raw rows arrive one iteration ahead of
// their conversion, which is one ahead of their use.
//
// The scores are scaled in fp32 behind the product (kRaw of the core).  Multiplying the query by scale * log2(e) beforehand
// would save a multiplication per score, 6 % of the time, but rounds the query once more: the output's error against 64 bits
// was 1.8 times that of one rounding at the end, now 1.4 times (what is left is the rounding of the probabilities).
#include "vqa_flash2.h"
#include "vqa_paged_attn.h"

namespace vqa {
namespace paged {
namespace chunk {

using flash::Geom;
using flash::u32x4_t;
using flash2::Scores;

constexpr int kBN = flash2::kBN;
constexpr int kRows = flash2::kBM;
constexpr int kWaves = 4;
static_assert(kBN == kKeyStep, "a key tile is a key step");

// e4m3: raw rows of one wave and tile pair (K of one tile, V of the one before): 16 rows each, then their exponents
template <int D>
struct Raw {
    static constexpr int kUnits = 16 * D / 1024;  // 1 KB each, per source
    static constexpr int kExp = 2 * 16 * D;
    static constexpr int kBytes = 2 * 16 * D + 64;
};

template <typename Tag, int D, bool kE4m3>
__global__ __launch_bounds__(kWaves * 64, 1) void chunk_kernel(AttnArgs a, Plan p) {
    typedef Geom<D> G;
    typedef flash2::Pipe<Tag, D, kWaves, true> Pipe;
    typedef typename Pipe::KDma KDma;
    typedef typename Pipe::VDma VDma;
    typedef typename Elem<Tag>::vec8 vec8;
    static_assert(KDma::kRowsPerWave == 16, "a wave's rows of a tile lie in one page");
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = __builtin_amdgcn_readfirstlane((int)(blockIdx.x % (unsigned)a.Hkv));
    const uint32_t lds0 = flash::lds_addr_of(smem);
    auto s_k = [&](int par) { return lds0 + (uint32_t)((par & 1) * G::kTileBytes); };
    auto s_v = [&](int par) { return lds0 + (uint32_t)((2 + (par & 1)) * G::kTileBytes); };

    KDma kd;
    VDma vd;
    if constexpr (!kE4m3) {
        kd.init(wave, lane, a.kp.sn / 2);
        vd.init(wave, lane, a.vp.sn / 2);
    }
    const char* k_head = a.kp.p + h * a.kp.sh;
    const char* v_head = a.vp.p + h * a.vp.sh;
    typedef Raw<D> RawG;
    auto s_raw = [&](int par) {
        return lds0 + (uint32_t)(4 * G::kTileBytes + ((par & 1) * kWaves + wave) * RawG::kBytes);
    };

    // e4m3, per lane (piece l % kPieces of row l / kPieces of a unit): byte of a unit's pieces in the pools, where its first
    // 16 widened bytes go in a tile, and the exponents' head (lane 0: keys, lane 1: values)
    constexpr int kPieces = D / 16, kUnitRows = 1024 / D;
    uint32_t k_raw = 0, v_raw = 0, k_dst = 0, v_dst = 0, e_step = 0;
    const uint8_t* e_head = nullptr;
    if constexpr (kE4m3) {
        const int r = lane / kPieces, c = lane % kPieces, row = 16 * wave + r;
        k_raw = (uint32_t)r * (uint32_t)a.kp.sn + (uint32_t)c * 16u;
        v_raw = (uint32_t)r * (uint32_t)a.vp.sn + (uint32_t)c * 16u;
        k_dst = (uint32_t)(row * G::kRowBytes + ((2 * c) ^ G::swz_k(row)) * 16);
        v_dst = (uint32_t)(row * G::kRowBytes + ((2 * c) ^ G::swz_v(row)) * 16);
        e_head = lane & 1 ? a.vp.e + h * a.vp.eh : a.kp.e + h * a.kp.eh;
        e_step = (uint32_t)(lane & 1 ? a.vp.ep : a.kp.ep);  // (the host has checked that it fits)
    }

    for_each_piece(a, p, lane,
                   [&](const Piece& u, int step, int n_steps, bool whole_tile, int slot_out) __attribute__((always_inline)) {
        const Seq& q = u.q;
        const int n_rows = q.n * a.G;  // of the sequence (fits 32 bits)
        const int row0 = u.tile * kRows + wave * flash2::kWaveRows;
        const int k_lo = step * kKeyStep;
        const int k_end = (int)min((int64_t)(step + n_steps) * kKeyStep, (int64_t)q.keys);
        const int n_iter = k_end > k_lo ? (k_end - k_lo + kBN - 1) / kBN : 0;

        // ---- pages: lane i holds where page tab0 + i begins, at this key head; `missing` says which are not there
        const int32_t* table = a.g.table + (int64_t)u.s * a.g.table_ss;
        const int in_page = (1 << a.g.page_shift) - 1;
        const uint32_t tile_pages = a.g.page_shift >= 6 ? 1u : a.g.page_shift == 5 ? 3u : 15u;  // a bit per page of a tile
        int64_t k_at = 0, v_at = 0;
        int tab = 0, tab0 = -0x40000000;
        uint64_t missing = 0;
        struct Place {
            const char *k, *v;  // this wave's first row of the tile
            int page;           // the page it lies in, and its row there
            uint32_t off;
            int last;           // its last row that is there, within 16 (at least 0)
            bool there;         // every page of the tile is there
        };
        // (t increases from call to call; kWhole: the tile has all 64 rows)
        auto place = [&](auto whole, int t) __attribute__((always_inline)) {
            constexpr bool kWhole = decltype(whole)::value;
            const int j0 = k_lo + t * kBN;
            const int c0 = j0 >> a.g.page_shift;
            if (c0 - tab0 >= 64) {  // (a block of entries begins with a tile, and 64 is a multiple of a tile's pages)
                tab0 = c0;
                const int e = c0 + lane < a.g.width ? table[c0 + lane] : -1;
                const bool ok = (unsigned)e < (unsigned)a.g.n_pages;
                missing = ~__builtin_amdgcn_ballot_w64(ok);
                tab = ok ? e : 0;  // (a page that is not there reads page 0; its keys are hidden)
                k_at = (int64_t)(uintptr_t)k_head + (int64_t)tab * a.kp.sp;
                v_at = (int64_t)(uintptr_t)v_head + (int64_t)tab * a.vp.sp;
            }
            Place x;
            const int jw = j0 + 16 * wave;
            const int j = kWhole || jw < k_end ? jw : (k_end - 1) & ~15;  // rows behind the end repeat the last one
            x.last = kWhole ? 15 : min(15, k_end - 1 - j);
            const int at = (j >> a.g.page_shift) - tab0;
            x.off = (uint32_t)(j & in_page);  // (a row's offset inside its page fits 32 bits)
            x.k = reinterpret_cast<const char*>((uintptr_t)lane64(k_at, at)) + x.off * (uint32_t)a.kp.sn;
            x.v = reinterpret_cast<const char*>((uintptr_t)lane64(v_at, at)) + x.off * (uint32_t)a.vp.sn;
            x.page = 0;
            if constexpr (kE4m3) x.page = __builtin_amdgcn_readlane(tab, at);
            x.there = ((uint32_t)(missing >> (c0 - tab0)) & tile_pages) == 0;
            return x;
        };
        typedef std::true_type Whole;
        typedef std::false_type Part;
        // which 16-row groups of tile t are there, bit by bit (rare)
        auto groups_there = [&](int t) {
            int bits = 0;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int j = k_lo + t * kBN + 16 * g;
                if (j < k_end) bits |= page_of(a.g, u.s, j) >= 0 ? 1 << g : 0;
            }
            return bits;
        };
        // a tile copy as a block: rows behind the end repeat the last one
        auto copy = [&](auto is_v, uint32_t tile, const char* rows, int last) __attribute__((always_inline)) {
            constexpr bool kV = decltype(is_v)::value;
            const int l = flash2::opaque_lane(lane);
            const uint32_t sn = (uint32_t)(kV ? a.vp.sn : a.kp.sn);
#pragma unroll
            for (int i = 0; i < KDma::kInstr; ++i) {
                const int r = i * G::kRowsPerInstr + l / G::kChunksPerRow;
                const int chunk = (l % G::kChunksPerRow) ^ (kV ? G::swz_v(16 * wave + r) : G::swz_k(16 * wave + r));
                flash::dma16_uniform(rows, (uint32_t)min(r, last) * sn + (uint32_t)chunk * 16u,
                                     tile + (uint32_t)((16 * wave + i * G::kRowsPerInstr) * G::kRowBytes));
            }
        };
        // ---- e4m3: raw rows in, widened rows out
        auto ask_raw = [&](auto is_v, auto whole, auto unit, uint32_t raw, const Place& x) __attribute__((always_inline)) {
            constexpr bool kV = decltype(is_v)::value;
            constexpr int j = decltype(unit)::value;
            const uint32_t sn = (uint32_t)(kV ? a.vp.sn : a.kp.sn);
            const char* rows = kV ? x.v : x.k;
            uint32_t off = kV ? v_raw : k_raw;
            if constexpr (decltype(whole)::value) {
                rows += j * kUnitRows * sn;
            } else {
                const int l = flash2::opaque_lane(lane);
                off = (uint32_t)min(j * kUnitRows + l / kPieces, x.last) * sn + (uint32_t)(l % kPieces) * 16u;
            }
            asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3"
                         :
                         : "s"(raw), "n"((kV ? 16 * D : 0) + j * 1024), "v"(off), "s"(rows)
                         : "memory", "scc");
        };
        // exponents of the 16 rows at kx (keys) and vx (values)
        auto ask_exp = [&](uint32_t raw, const Place& kx, const Place& vx) __attribute__((always_inline)) {
            const int l = flash2::opaque_lane(lane);
            const uint8_t* src = e_head + (uint64_t)(uint32_t)(l & 1 ? vx.page : kx.page) * e_step + (l & 1 ? vx.off : kx.off);
            if (l < 2) flash::dma16(src, raw + RawG::kExp);
        };
        struct Unit {
            u32x4_t x;
            uint32_t e;
        };
        typedef const __attribute__((address_space(3))) u32x4_t* lds16_in;
        typedef __attribute__((address_space(3))) u32x4_t* lds16_out;
        typedef const __attribute__((address_space(3))) uint8_t* lds8_in;
        // (rows behind the last one repeat it, so its exponent goes with them: what stands behind it may be anything)
        auto read_unit = [&](bool v, int j, uint32_t raw, int last) __attribute__((always_inline)) {
            const int l = flash2::opaque_lane(lane);
            Unit r;
            r.x = *(lds16_in)(uintptr_t)(raw + (uint32_t)((v ? 16 * D : 0) + j * 1024 + l * 16));
            r.e = *(lds8_in)(uintptr_t)(raw + (uint32_t)(RawG::kExp + (v ? 16 : 0) + min(j * kUnitRows + l / kPieces, last)));
            return r;
        };
        // where the unit's first 16 bytes go (the second 16 lie at that address ^ 16): 8 rows on, the key tile's XOR has
        // another bit, the value tile's has not
        auto unit_dst = [&](bool v, int j, uint32_t tile) __attribute__((always_inline)) {
            static_assert(RawG::kUnits <= 2, "the XOR of a third unit is not looked after");
            return tile + (v ? v_dst : k_dst ^ (uint32_t)(j * 128)) + (uint32_t)(j * kUnitRows * G::kRowBytes);
        };
        auto widen_unit = [&](const Unit& r, uint32_t dst) __attribute__((always_inline)) {
            const float f = factor_of((int)r.e);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint2 p0 = widen4<Tag>(r.x[2 * e], f), p1 = widen4<Tag>(r.x[2 * e + 1], f);
                *(lds16_out)(uintptr_t)(dst ^ (uint32_t)(16 * e)) = u32x4_t{p0.x, p0.y, p1.x, p1.y};
            }
        };
        auto widen_block = [&](bool v, uint32_t raw, uint32_t tile, int last) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < RawG::kUnits; ++j) widen_unit(read_unit(v, j, raw, last), unit_dst(v, j, tile));
        };
        typedef std::false_type K;
        typedef std::true_type V;

        // ---- rows of this lane: what they see; the wave's common part
        int tok[2];  // new token of each of the lane's two rows
        flash2::Wave<Tag, D> w;
        w.init();
        w.c = a.scale_log2e;
        // (the queries are asked for before the table and the first tiles, which depend on it)
        const int t_first = min(row0, n_rows - 1) / a.G, t_last = min(row0 + flash2::kWaveRows - 1, n_rows - 1) / a.G;
        const int all_hi = visible(a, q, t_first).hi, all_lo = visible(a, q, t_last).lo;
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
            const int r = min(row0 + qb * 32 + (lane & 31), n_rows - 1);  // rows past the end are computed, never stored
            const int t = r / a.G, g = r - t * a.G;
            tok[qb] = t;
            const uint16_t* src = a.q + (int64_t)(q.q0 + t) * a.q_st + (int64_t)(h * a.G + g) * a.q_sh + (lane >> 5) * 8;
#pragma unroll
            for (int kk = 0; kk < G::kKSteps; ++kk) w.q[qb].f[kk] = *reinterpret_cast<const vec8*>(src + kk * 16);
        }
        Place now = {nullptr, nullptr, 0, 0, 0, true}, next = now, after = now;
        if (kE4m3 && n_iter > 0) {
            auto ask_all = [&](auto is_v, uint32_t raw, const Place& x) __attribute__((always_inline)) {
                flash2::static_for<RawG::kUnits>([&](auto J) { ask_raw(is_v, Part(), J, raw, x); });
            };
            now = place(Part(), 0);
            ask_all(K(), s_raw(0), now);
            ask_all(V(), s_raw(0), now);
            ask_exp(s_raw(0), now, now);
            next = now;
            if (n_iter > 1) {
                next = place(Part(), 1);
                ask_all(K(), s_raw(1), next);
                ask_exp(s_raw(1), next, next);
            }
            flash::wait_tile_loads();
            asm volatile("" ::: "memory");
            widen_block(false, s_raw(0), s_k(0), now.last);
            widen_block(true, s_raw(0), s_v(0), now.last);
            widen_block(false, s_raw(1), s_k(1), next.last);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            after = next;
            if (n_iter > 1) ask_all(V(), s_raw(0), next);
            if (n_iter > 2) {
                after = place(Part(), 2);
                ask_all(K(), s_raw(0), after);
            }
            ask_exp(s_raw(0), after, next);
        }
        if (!kE4m3 && n_iter > 0) {
            now = place(Part(), 0);
            copy(K(), s_k(0), now.k, now.last);
            copy(V(), s_v(0), now.v, now.last);
            next = now;
            if (n_iter > 1) {
                next = place(Part(), 1);
                copy(K(), s_k(1), next.k, next.last);
            }
        }
#pragma unroll
        for (int qb = 0; qb < 2; ++qb)
#pragma unroll
            for (int kk = 0; kk < G::kKSteps; ++kk) {
                u32x4_t x = __builtin_bit_cast(u32x4_t, w.q[qb].f[kk]);
                asm volatile("" : "+a"(x));  // (only ever MFMA operands: they live in AccVGPRs)
                w.q[qb].f[kk] = __builtin_bit_cast(vec8, x);
            }

        Scores s_even, s_odd;
        typename Pipe::Frags kf, vf;
        float mx[2] = {-INFINITY, -INFINITY};
        auto mask_tile = [&](Scores& sn, int t, bool there) __attribute__((always_inline)) {
            const int n0 = k_lo + t * kBN;
            if (there && n0 + kBN <= all_hi && n0 >= all_lo && t < n_iter) return;  // (wave-uniform)
            flash2::mfma_settle(sn);
            const int half = flash2::opaque_lane(lane) >> 5;
            const int bits = t < n_iter ? (there ? 15 : groups_there(t)) : 0;
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                const Range x = visible(a, q, tok[qb]);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = n0 + kb * 32 + flash::key_of_reg(r, half);
                        const bool seen = j < x.hi && j >= x.lo && ((bits >> (2 * kb + (r >> 3))) & 1);
                        sn.s[qb][kb][r] = seen ? sn.s[qb][kb][r] : -INFINITY;
                    }
            }
        };
        const typename Pipe::TileRequest no_req{nullptr, 0};

        if (n_iter > 0) {
            if constexpr (!kE4m3) flash::wait_tile_loads();
            __syncthreads();
            Pipe::k_head(kf, s_k(0), lane);
            Pipe::template score_phase<true, false, false, false>(w, s_even, kf, s_odd, vf, 0u, lane, kd, no_req, vd, no_req);
            mask_tile(s_even, 0, now.there);
            Pipe::template pv_phase<false, true>(w, vf, s_odd, s_even, mx);
        }
        // Iteration t finishes tile t and scores tile t + 1; it requests K(t + 2) and V(t + 1).  `next` is the place of tile
        // t + 1 when it begins.
        auto iteration = [&](auto t_is_odd, auto ride, int t) __attribute__((always_inline)) {
            constexpr int par = decltype(t_is_odd)::value ? 1 : 0;
            constexpr bool kRide = decltype(ride)::value;
            Scores& sc = par ? s_odd : s_even;
            Scores& sn = par ? s_even : s_odd;
            flash::wait_tile_loads();
            __syncthreads();  // K(t + 1) and V(t) are complete; every wave is done with K(t) and V(t - 1)
            Pipe::k_head(kf, s_k(par + 1), lane);
            typename Pipe::TileRequest kr = no_req, vr = no_req;
            const bool there = next.there;
            if constexpr (kRide) {
                vr.rows = next.v;
                vr.lds = VDma::lds_of_wave(s_v(par + 1), wave);
                next = place(Whole(), t + 2);
                kr.rows = next.k;
                kr.lds = KDma::lds_of_wave(s_k(par), wave);
            } else {
                if (t + 1 < n_iter) copy(V(), s_v(par + 1), next.v, next.last);
                if (t + 2 < n_iter) {
                    next = place(Part(), t + 2);
                    copy(K(), s_k(par), next.k, next.last);
                }
            }
            Pipe::update_max(w, mx, sc);
            Pipe::template score_phase<true, true, true, kRide>(w, sn, kf, sc, vf, s_v(par), lane, kd, kr, vd, vr);
            mask_tile(sn, t + 1, there);
            mx[0] = mx[1] = -INFINITY;
            Pipe::template pv_phase<true, true>(w, vf, sc, sn, mx);
        };
        // e4m3: `next` and `after` are the places of tiles t + 1 and t + 2; the raw rows of K(t + 2) and V(t + 1) have arrived
        // when iteration t begins and are widened in it, those of K(t + 3) and V(t + 2) are requested.
        auto iteration8 = [&](auto t_is_odd, auto whole, int t) __attribute__((always_inline)) {
            constexpr int par = decltype(t_is_odd)::value ? 1 : 0;
            Scores& sc = par ? s_odd : s_even;
            Scores& sn = par ? s_even : s_odd;
            flash::wait_tile_loads();
            __syncthreads();
            Pipe::k_head(kf, s_k(par + 1), lane);
            const bool there = next.there;
            const Place v_of = after;  // tile t + 2
            Place k_of = after;
            constexpr bool kWhole = decltype(whole)::value;  // tiles t + 2 and t + 3 have all 64 rows
            const bool more_v = kWhole || t + 2 < n_iter, more_k = kWhole || t + 3 < n_iter;
            if (more_k) k_of = place(whole, t + 3);
            const uint32_t raw_in = s_raw(par), raw_out = s_raw(par + 1);
            const int k_last = kWhole ? 15 : after.last, v_last = kWhole ? 15 : next.last;  // of K(t + 2) and V(t + 1)
            Unit unit = read_unit(false, 0, raw_in, k_last), coming = unit;
            uint32_t dst = 0;
            float f = 0.f;
            u32x4_t half;
            Pipe::update_max(w, mx, sc);
            constexpr int kU = 2 * RawG::kUnits;  // units in the order K .. V ..
            static_assert(Pipe::kScoreSlots == 8 * kU, "a unit takes eight slots");
            Pipe::template score_phase<true, true, true, false>(
                w, sn, kf, sc, vf, s_v(par), lane, kd, no_req, vd, no_req, [&](auto I) __attribute__((always_inline)) {
                    constexpr int i = decltype(I)::value, U = i / 8, s = i % 8;
                    constexpr bool v = U >= RawG::kUnits;
                    constexpr int j = U % RawG::kUnits;
                    if constexpr (s == 0) {
                        dst = unit_dst(v, j, v ? s_v(par + 1) : s_k(par));
                        f = factor_of((int)unit.e);
                        flash2::pin(f);
                    }
                    if constexpr (s == 1 || s == 2 || s == 4 || s == 5) {
                        constexpr int word = s < 3 ? s - 1 : s - 2;
                        const uint2 p = widen4<Tag>(unit.x[word], f);
                        half[2 * (word & 1)] = p.x, half[2 * (word & 1) + 1] = p.y;
                    }
                    if constexpr (s == 3) *(lds16_out)(uintptr_t)dst = half;
                    if constexpr (s == 6) *(lds16_out)(uintptr_t)(dst ^ 16u) = half;
                    if constexpr (s == 4 && U + 1 < kU) {
                        constexpr int n = U + 1;
                        coming = read_unit(n >= RawG::kUnits, n % RawG::kUnits, raw_in, n >= RawG::kUnits ? v_last : k_last);
                    }
                    if constexpr (s == 7) {
                        unit = coming;
                        if constexpr (v) {
                            if (more_v) ask_raw(V(), whole, std::integral_constant<int, j>{}, raw_out, v_of);
                        } else {
                            if (more_k) ask_raw(K(), whole, std::integral_constant<int, j>{}, raw_out, k_of);
                        }
                        if constexpr (U == kU - 1)
                            if (more_v) ask_exp(raw_out, k_of, v_of);
                    }
                });
            mask_tile(sn, t + 1, there);
            next = v_of, after = k_of;
            mx[0] = mx[1] = -INFINITY;
            Pipe::template pv_phase<true, true>(w, vf, sc, sn, mx);
        };
        int t = 0;
        const int n_whole = (k_end - k_lo) / kBN;  // tiles with all 64 rows
        if constexpr (kE4m3) {
            for (; t + 4 < n_whole; t += 2) {
                iteration8(std::false_type{}, Whole(), t);
                iteration8(std::true_type{}, Whole(), t + 1);
            }
            for (; t < n_iter; t += 2) {
                iteration8(std::false_type{}, Part(), t);
                if (t + 1 < n_iter) iteration8(std::true_type{}, Part(), t + 1);
            }
        } else {
            for (; t + 3 < n_whole; t += 2) {
                iteration(std::false_type{}, std::true_type{}, t);
                iteration(std::true_type{}, std::true_type{}, t + 1);
            }
            for (; t < n_iter; t += 2) {
                iteration(std::false_type{}, std::false_type{}, t);
                if (t + 1 < n_iter) iteration(std::true_type{}, std::false_type{}, t + 1);
            }
        }
        Pipe::settle_o(w);
        __syncthreads();  // no wave reads tiles any more

        // ---- results.  A row that came out as infinity or NaN may have met one in a value it does not see (0 * inf): it is
        // done again, key by key.
        const int half = lane >> 5, n = lane & 31;
        uint64_t bad = 0;
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
            const float l = flash2::join_halves_sum(w.l[qb][0] + w.l[qb][1]);
            const float m = w.m[qb] * w.c;  // (-inf stays -inf)
            const int r = row0 + qb * 32 + n;
            float probe = l;
#pragma unroll
            for (int db = 0; db < G::kDBlocks; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) probe += w.o[qb][db][i] * 0.f;
            const uint64_t vote = __builtin_amdgcn_ballot_w64(!(probe < INFINITY) && r < n_rows);
            bad |= ((vote | (vote >> 32)) & 0xffffffffull) << (32 * qb);
            if (whole_tile) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                char* dst = smem + wave * Pipe::kStoreBytes + (qb * 32 + n) * Pipe::kStoreRowBytes;
#pragma unroll
                for (int db = 0; db < G::kDBlocks; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<uint2*>(dst + (db * 32 + 8 * g + 4 * half) * 2) =
                            make_uint2(Elem<Tag>::pack2(w.o[qb][db][4 * g] * inv, w.o[qb][db][4 * g + 1] * inv),
                                       Elem<Tag>::pack2(w.o[qb][db][4 * g + 2] * inv, w.o[qb][db][4 * g + 3] * inv));
                if (a.lse != nullptr && half == 0 && r < n_rows) {
                    const int t = r / a.G;
                    a.lse[(int64_t)(q.q0 + t) * a.Hq + h * a.G + r - t * a.G] = l == 0.f ? -INFINITY : m + fast_log2(l);
                }
            } else if (r < n_rows) {
                const int64_t at = ((int64_t)slot_out * a.Hkv + h) * kRows + wave * flash2::kWaveRows + qb * 32 + n;
#pragma unroll
                for (int db = 0; db < G::kDBlocks; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<float4*>(p.o + at * D + db * 32 + 8 * g + 4 * half) = make_float4(
                            w.o[qb][db][4 * g], w.o[qb][db][4 * g + 1], w.o[qb][db][4 * g + 2], w.o[qb][db][4 * g + 3]);
                if (half == 0) p.ml[at * 2] = m, p.ml[at * 2 + 1] = l;
            }
        }
        if (whole_tile) {
            wave_lds_sync();
            constexpr int kLanesPerRow = G::kRowBytes / 16, kRowsPerInstr = 64 / kLanesPerRow;
            const int c = lane % kLanesPerRow;
            const int t0 = row0 / a.G, g0 = row0 - t0 * a.G;
            const float inv_g = 1.f / (float)a.G;
#pragma unroll
            for (int i = 0; i < flash2::kWaveRows / kRowsPerInstr; ++i) {
                const int in = i * kRowsPerInstr + lane / kLanesPerRow, r = row0 + in;
                const char* src = smem + wave * Pipe::kStoreBytes + in * Pipe::kStoreRowBytes + c * 16;
                const uint2 x = *reinterpret_cast<const uint2*>(src), y = *reinterpret_cast<const uint2*>(src + 8);
                if (r < n_rows) {
                    // (small numbers: exact in fp32, and half a step away from the next whole one)
                    const int z = g0 + in, dt = (int)(((float)z + 0.5f) * inv_g);
                    *reinterpret_cast<uint4*>(a.out + (int64_t)(q.q0 + t0 + dt) * a.o_st + (int64_t)(h * a.G + z - dt * a.G) * a.o_sh +
                                              c * 8) = make_uint4(x.x, x.y, y.x, y.y);
                }
            }
        }
        for (; bad; bad &= bad - 1) {
            const int in = __builtin_ctzll(bad), r = row0 + in, t = r / a.G, hq = h * a.G + r - t * a.G;
            const Range x = visible(a, q, t);
            RowState<D> st;
            row_by_lanes<Tag, D, kE4m3>(a, u.s, h, a.q + (int64_t)(q.q0 + t) * a.q_st + (int64_t)hq * a.q_sh,
                                        max(k_lo, x.lo), min(k_end, x.hi), st, lane);
            if (whole_tile) {
                store_row<Tag, D>(a, st, q.q0 + t, hq, lane);
            } else {
                const int64_t at = ((int64_t)slot_out * a.Hkv + h) * kRows + wave * flash2::kWaveRows + in;
#pragma unroll
                for (int e = 0; e < D / 64; ++e) p.o[at * D + lane * (D / 64) + e] = st.o[e];
                if (lane == 0) p.ml[at * 2] = st.m, p.ml[at * 2 + 1] = st.l;
            }
        }
        __syncthreads();  // the staging area is free for the next piece's tiles
    });
}

template <typename Tag, int D, bool kE4m3>
int launch(const AttnArgs& a, const Plan& p, int64_t grid, int dev, hipStream_t stream) {
    constexpr int tiles = 4 * Geom<D>::kTileBytes + (kE4m3 ? 2 * kWaves * Raw<D>::kBytes : 0);
    constexpr int stage = kWaves * flash2::Pipe<Tag, D, kWaves, true>::kStoreBytes;
    constexpr int bytes = tiles > stage ? tiles : stage;
    if (bytes > 64 * 1024)
        if (int rc = raise_lds<chunk_kernel<Tag, D, kE4m3>>(dev, bytes)) return rc;
    chunk_kernel<Tag, D, kE4m3><<<dim3((unsigned)grid), kWaves * 64, bytes, stream>>>(a, p);
    return launch_status();
}

}  // namespace chunk

template <typename Tag>
int launch_chunk(const AttnArgs& a, const Plan& p, int D, bool e4m3, int64_t grid, int dev, hipStream_t stream) {
    if (D == 128)
        return e4m3 ? chunk::launch<Tag, 128, true>(a, p, grid, dev, stream) : chunk::launch<Tag, 128, false>(a, p, grid, dev, stream);
    return e4m3 ? chunk::launch<Tag, 64, true>(a, p, grid, dev, stream) : chunk::launch<Tag, 64, false>(a, p, grid, dev, stream);
}
template int launch_chunk<bf16_tag>(const AttnArgs&, const Plan&, int, bool, int64_t, int, hipStream_t);
template int launch_chunk<f16_tag>(const AttnArgs&, const Plan&, int, bool, int64_t, int, hipStream_t);

}  // namespace paged
}  // namespace vqa
