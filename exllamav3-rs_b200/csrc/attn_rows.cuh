// Attention over spans of the cache for sequences of few rows: at most 16 (query, head) rows per kv head, a decode row with its sibling
// heads or a few of them.
//
// Bound by HBM: every visible key and value is read once, and the two products are far below what mma.sync gives.  So the work is a
// stream: all sequences' key tiles, head group after head group, stand in one line, and every CTA takes an equal part of it, whatever the
// lengths (a CTA per SM; the parts are found from the lengths by each CTA itself, so there is no list to build in front).  A
// producer warp runs ahead through a ring of six tiles and over the borders of sequences, so that the end of one costs no loads.
//
// A tile is 32 KB of keys and values, for four warps: HW = 4 heads side by side and 16 keys, a head per warp, where the kv heads come in
// fours - 1 KB of every token in one piece, and no warp needs another - else one head and 64 keys, 16 per warp, which meet at the end of
// a unit.  (One head and 64 keys of 8: 128 rows over windows of 4096, 256-byte pieces, 262 us, where as it is it took 191; 193 to 210 us on the
// machines it was timed on since, 5.6 to 6.1 TB/s.)
//
// A sequence and head group whose tiles fall to several CTAs goes through partial sums, which the one that arrives last adds up in the
// order of the tiles: results do not depend on who that is.  Keys of a tile that no row sees are not loaded where they fill a group of 16,
// and masked in both products where not (a masked key's value may be NaN).
#pragma once
#include <cuda.h>
#include "attn_span.cuh"
#include "attn_tc_ops.cuh"
#include "async_copy.cuh"

namespace exl3 {

constexpr int AR_ROWS = 16, AR_STAGES = 6, AR_WARPS = 4;
constexpr int AR_THREADS = (AR_WARPS + 1) * 32;
constexpr int AR_STAGE = 32768;                         // keys and values of a tile
constexpr int AR_MS = SPAN_PART;
constexpr int AR_MAX_BSZ = 1024;                        // sequences of a launch: their tile counts are summed in shared memory
constexpr int AR_SNAP = 6;                              // a part ends with a unit that would end so many tiles from there
constexpr int AR_UNITS = AR_STAGES + 1;                 // unit descriptors: the producer is at most AR_STAGES tiles, so units, ahead

constexpr int AR_PREFIX = 1 << 30;                      // bit of a tile that is read for a prefix

struct ArUnit { int b, hg, row_base, ql, cached, key_lo, group, whole, slot, c0, pieces, tiles; };

template <int HW>
struct ArCfg {
    static constexpr int KW = AR_WARPS / HW, TK = 16 * KW;                          // warps that share a head's keys, keys of a tile
    static constexpr int HALF = TK * 128, HEAD = 2 * HALF;                          // bytes of a 64-dim half of a head, rows of 128 bytes in the 128-byte swizzle
    static constexpr int OFF_MERGE = AR_STAGES * AR_STAGE;                          // KW > 1: rows of every head
    static constexpr int OFF_ML = OFF_MERGE + (KW > 1 ? HW * AR_ROWS * AR_MS * 4 : 0);
    static constexpr int OFF_SUM = OFF_ML + AR_WARPS * AR_ROWS * 8;
    static constexpr int OFF_UNIT = OFF_SUM + (AR_MAX_BSZ + 4) * 4;
    static constexpr int OFF_BAR = OFF_UNIT + AR_UNITS * (int)sizeof(ArUnit);
    // full[stages], empty[stages], meet; then the tile of every stage
    static constexpr int OFF_TILE = OFF_BAR + (2 * AR_STAGES + 1) * 8;
    static constexpr int BYTES = OFF_TILE + AR_STAGES * 4 + 16 + 1024;
    static_assert(HW * HEAD * 2 == AR_STAGE, "a tile");
    static_assert(BYTES + 1024 + 64 <= EXL3_SM_SMEM, "a CTA per SM");
    static_assert(OFF_ML % 8 == 0 && OFF_BAR % 8 == 0, "alignment");
};

template <int N> struct ArInt { static constexpr int value = N; };

struct ArMaps { CUtensorMap k, v, k16, v16; };          // boxes of a tile, and of 16 tokens of one half of one head

struct ArParams {
    SpanArgs a;
    int b0, bsz;                                        // sequences of this launch
    int min_share;                                      // tiles that a CTA takes at least
    float* partial;                                     // [2 * CTAs][HW][16][AR_MS]
    int* counters;                                      // [CTAs][4], zero between calls
    int* status;
    float* rest;                                        // [rows][nq][AR_MS] partial sums of sequences that a prefix is added to
    int first;                                          // nothing of this call is in front of the launch
};

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4, uint64_t* bar)
{
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar)) : "memory");
}

// ALONE: prefixes are read here too, through their own table, by each sequence.  (A kernel of its own: with both kinds of tiles in every loop
// 128 rows over windows of 4096 took 210 us for 193, a row over 1024 13.4 for 12.6.)  BESIDE: the other kernel runs at the same time.
template <int HW, bool ALONE, bool BESIDE>
__global__ void __launch_bounds__(AR_THREADS, 1) attn_rows_kernel(const __grid_constant__ ArMaps maps, const ArParams p, int early)
{
    using Cfg = ArCfg<HW>;
    constexpr int KW = Cfg::KW, TK = Cfg::TK, PER_PAGE = EXL3_PAGE / TK;
    if (p.first) pdl_enter_first(early);
    else asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint8_t smem_unaligned[];
    uint8_t* smem = smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u);
    float2* ml = reinterpret_cast<float2*>(smem + Cfg::OFF_ML);                     // [warp][row]
    int* sum = reinterpret_cast<int*>(smem + Cfg::OFF_SUM);                         // [bsz + 1] first tile of every sequence, per head group
    ArUnit* units = reinterpret_cast<ArUnit*>(smem + Cfg::OFF_UNIT);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
    uint64_t* empty = full + AR_STAGES;
    uint64_t* meet = empty + AR_STAGES;
    int* tile_of = reinterpret_cast<int*>(smem + Cfg::OFF_TILE);                    // key tile in a stage, -1: none of its keys exist
    __shared__ int s_last;
    __shared__ SpanLoad loads[BESIDE ? AR_WARPS + 1 : 1];

    const SpanArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.nq / a.nkv, n_hg = a.nkv / HW;
    if (tid == 0) {
        for (int i = 0; i < AR_STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], AR_WARPS); }
        mbar_init(meet, AR_WARPS);
        mbar_fence_init();
    }
    // a sequence's tiles, at least one if it has rows of this kernel (their output is written)
    auto tiles_of = [&](int b) -> int {
        const SpanSeq s = span_seq(a, b);
        if (s.ql == 0 || s.ql * G > AR_ROWS) return 0;
        const int len = span_group(a, b, s.cached).len;
        const SpanTiles t = span_tiles<TK>(a, s.cached, s.cached + s.ql - 1, len);
        return max((ALONE ? (len + TK - 1) / TK : 0) + t.sink + t.near, 1);
    };
    SpanLoad load = {0, 0};
    for (int b = tid; b < p.bsz; b += AR_THREADS) {
        sum[b] = tiles_of(p.b0 + b);
        if (BESIDE) span_load(a, b, AR_ROWS, load);
    }
    if (BESIDE) span_load_put(loads, warp, load, lane);
    __syncthreads();
    if (warp == 0) {
        int before = 0;
        for (int b = lane; b - lane < p.bsz; b += 32) {
            const int own = b < p.bsz ? sum[b] : 0;
            int v = own;
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += u; }
            if (b < p.bsz) sum[b] = before + v - own;
            before += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) sum[p.bsz] = before;
    }
    __syncthreads();
    // this CTA's part [f0, f1) of the line of all tiles: sequence, head group, tile.  (A 64-bit division is a quarter of a microsecond of every
    // CTA's start: what fits in 32 bits is divided there.)
    auto quotient = [](long long x, int y) -> long long { return x >> 32 ? x / y : (long long)((unsigned)x / (unsigned)y); };
    const long long F = (long long)sum[p.bsz] * n_hg;
    const int ctas = BESIDE ? max(span_few_sms(a, loads, AR_WARPS + 1), 1) : gridDim.x;
    const long long share = max(quotient(F + ctas - 1, ctas), (long long)p.min_share);
    const int c = blockIdx.x, snap = (int)min((long long)AR_SNAP, share / 4);
    auto sequence_of = [&](long long f) -> int {            // the one with tile f: sum[b] * n_hg <= f < sum[b + 1] * n_hg
        const long long per_group = quotient(f, n_hg);
        int lo = 0, hi = p.bsz;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (sum[mid] <= per_group) lo = mid; else hi = mid; }
        return lo;
    };
    // Where part c begins.  A cut unit costs some 5 us, its partial sums' way through memory: parts end with a unit that ends near by.
    auto begin_of = [&](int c) -> long long {
        const long long f = c * share;
        if (c == 0 || f >= F) return min(f, F);
        const int b = sequence_of(f), n = sum[b + 1] - sum[b];
        const long long in = f - (long long)sum[b] * n_hg;
        const int from = (int)(in - quotient(in, n) * n);
        return from <= snap && from <= n - from ? f - from : n - from <= snap ? f + (n - from) : f;
    };
    const long long begins = begin_of(c + (lane & 1));      // side by side
    const long long f0 = __shfl_sync(0xffffffffu, begins, 0), f1 = __shfl_sync(0xffffffffu, begins, 1);
    if (f0 >= f1) {
        if (!p.first) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    // the last parts that do not begin behind a unit's first and last tile: the two parts around each, and itself, side by side
    auto parts_of = [&](long long first, long long last, int& c0, int& c1) {
        const long long f = lane & 4 ? last : first;
        const int k = (int)(share >> 31 ? f / share : quotient(f, (int)share)) - 1 + (lane & 3);
        const unsigned in = __ballot_sync(0xffffffffu, (lane & 3) < 3 && k >= 0 && begin_of(k) <= f);
        c0 = __shfl_sync(0xffffffffu, k, 31 - __clz(in & 0x0fu));
        c1 = __shfl_sync(0xffffffffu, k, 31 - __clz(in & 0xf0u));
    };

    if (warp == AR_WARPS) {
        // ===== producer: the whole warp walks, lane 0 issues; lane i holds the block table's entry page0 + i
        int it = 0, n_unit = 0;
        long long f = f0;
        int b = sequence_of(f0);
        bool ok = true;
        SpanSeq s = {0, 0, 0};
        SpanTiles t = {};
        SpanGroup grp = {-1, 0, 0};
        int have = -1, page0 = 0, entry = 0, n_pre = 0;
        while (f < f1 && ok) {
            while ((long long)sum[b + 1] * n_hg <= f) ++b;
            const int n = sum[b + 1] - sum[b];
            const long long in = f - (long long)sum[b] * n_hg;
            const int hg = (int)quotient(in, n), from = (int)(in - (long long)hg * n);
            const int upto = (int)min((long long)n, from + (f1 - f));
            const int gb = p.b0 + b;
            if (have != b) {
                s = span_seq(a, gb);
                grp = span_group(a, gb, s.cached);
                t = span_tiles<TK>(a, s.cached, s.cached + s.ql - 1, grp.len);
                n_pre = ALONE ? (grp.len + TK - 1) / TK : 0;
                have = b;
            }
            page0 = -64;
            const long long u0 = f - from;
            for (int i = from; i < upto; ++i, ++it) {
                const int stage = it % AR_STAGES;
                const bool pre = ALONE && i < n_pre;
                const int own = i - n_pre, kt = pre ? i : t.sink + t.near == 0 ? -1 : own < t.sink ? own : t.first + (own - t.sink);
                const int32_t* bt = a.block_table + (size_t)(pre ? grp.first : gb) * a.pps;
                if (ALONE && i == n_pre) page0 = -64;
                int page = -1;
                if (kt >= 0) {
                    const int pg = kt / PER_PAGE;
                    if (pg < page0 || pg >= page0 + 32) { page0 = pg; entry = pg + lane < a.pps ? bt[pg + lane] : -1; }
                    page = __shfl_sync(0xffffffffu, entry, pg - page0);
                    if (page >= a.pages) page = -1;
                }
                if (it >= AR_STAGES && !mbar_wait_sleep_warp(&empty[stage], ((it / AR_STAGES) - 1) & 1)) { ok = false; break; }
                // what a cut unit's partial sums need is found under the copies of its tiles, and read behind the last one
                const bool cut = i == upto - 1 && !(from == 0 && upto == n);
                int c0 = 0, c1 = 0;
                if (cut) parts_of(u0, u0 + n - 1, c0, c1);
                if (lane == 0) {
                    if (cut) { units[n_unit % AR_UNITS].c0 = c0; units[n_unit % AR_UNITS].pieces = c1 - c0 + 1; }
                    if (i == from) {
                        ArUnit& u = units[n_unit % AR_UNITS];
                        u.b = gb; u.hg = hg; u.row_base = s.row_base; u.ql = s.ql; u.cached = s.cached; u.key_lo = grp.len; u.group = ALONE ? -1 : grp.g;
                        u.whole = from == 0 && upto == n;
                        u.slot = 2 * c + (from == 0 ? 1 : 0);
                        u.tiles = upto - from;
                    }
                    tile_of[stage] = page < 0 ? -1 : pre ? kt | AR_PREFIX : kt;
                    if (page < 0) mbar_arrive(&full[stage]);
                    else {
                        // groups of 16 keys with one that some row sees
                        const int k0 = kt * TK, tok = k0 & (EXL3_PAGE - 1);
                        int g0 = 0, g1 = KW;
                        if constexpr (KW > 1) {
                            const int hi = min(TK, (pre ? grp.len : own < t.sink ? min(a.sinks, t.end) : t.end) - k0);
                            const int lo = pre || own < t.sink || a.sinks > k0 ? 0 : max(0, t.lo - k0);
                            g0 = lo >> 4; g1 = (hi + 15) >> 4;
                        }
                        uint8_t* st = smem + stage * AR_STAGE;
                        mbar_expect_tx(&full[stage], (g1 - g0) * (AR_STAGE / KW));
                        if (g1 - g0 == KW) {
                            tma_load_5d(st, &maps.k, 0, tok, 0, hg * HW, page, &full[stage]);
                            tma_load_5d(st + AR_STAGE / 2, &maps.v, 0, tok, 0, hg * HW, page, &full[stage]);
                        } else
                            for (int g = g0; g < g1; ++g)
                                for (int h = 0; h < 2 * HW; ++h) {
                                    uint8_t* at = st + h * Cfg::HALF + g * 2048;
                                    tma_load_5d(at, &maps.k16, 0, tok + 16 * g, h & 1, hg * HW + (h >> 1), page, &full[stage]);
                                    tma_load_5d(at + AR_STAGE / 2, &maps.v16, 0, tok + 16 * g, h & 1, hg * HW + (h >> 1), page, &full[stage]);
                                }
                    }
                }
                __syncwarp();
            }
            f = u0 + upto; ++n_unit;
        }
        if (!ok) {
            // nobody takes the tiles any more: out only when the copies in flight have landed
            for (int k = max(0, it - AR_STAGES); k < it; ++k) mbar_wait_sleep_warp(&full[k % AR_STAGES], (k / AR_STAGES) & 1);
            if (lane == 0) atomicExch(p.status, 3);
        }
        return;
    }

    // ===== four warps: head wh of the group, keys 16 wk .. of every tile
    const int wh = warp / KW, wk = warp % KW;
    uint32_t meet_phase = 0;
    auto rendezvous = [&]() -> bool {                   // bounded, unlike a named barrier: a warp may have left through a time-out
        __syncwarp();
        if (lane == 0) mbar_arrive(meet);
        const bool r = mbar_wait_warp(meet, meet_phase);
        meet_phase ^= 1;
        return r;
    };
    const int g = lane >> 2, t4 = lane & 3;
    bool ok = true;
    int it = 0, n_unit = 0;
    for (long long f = f0; f < f1 && ok; ++n_unit) {
        if (!mbar_wait_warp(&full[it % AR_STAGES], (it / AR_STAGES) & 1)) { ok = false; break; }
        ArUnit u = units[n_unit % AR_UNITS];
        f += u.tiles;
        const int n_rows = u.ql * G, kvh = u.hg * HW + wh;
        int lo[2], hi[2];
        bool valid[2];
        uint32_t qf[8][4];
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = g + 8 * h, qi = row / G, pos = u.cached + qi;
            valid[h] = row < n_rows;
            hi[h] = min(max(pos + 1, 0), a.pps * EXL3_PAGE);
            lo[h] = max(u.key_lo, a.window > pos ? 0 : pos - a.window + 1);
            const half* qp = a.q + ((size_t)(u.row_base + qi) * a.nq + kvh * G + (row - qi * G)) * 128;
            #pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                qf[ks][h]     = valid[h] ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + 2 * t4) : 0u;
                qf[ks][h + 2] = valid[h] ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + 8 + 2 * t4) : 0u;
            }
        }
        // what all rows see, and what any row sees
        const int p_last = u.cached + u.ql - 1;
        const int all_hi = min(max(u.cached + 1, 0), a.pps * EXL3_PAGE), any_hi = min(max(p_last + 1, 0), a.pps * EXL3_PAGE);
        const int any_lo = max(u.key_lo, a.window > u.cached ? 0 : u.cached - a.window + 1);
        const int all_lo = max(u.key_lo, a.window > p_last ? 0 : p_last - a.window + 1);

        float o_acc[16][4];
        #pragma unroll
        for (int i = 0; i < 16; ++i) { o_acc[i][0] = o_acc[i][1] = o_acc[i][2] = o_acc[i][3] = 0.f; }
        float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
        // two tiles at a time where there are two: most of a step is latency, of which they have one
        for (int i = 0; i < u.tiles; i += 2) {
            const bool two = i + 1 < u.tiles;
            const int st0 = it % AR_STAGES, st1 = two ? (it + 1) % AR_STAGES : st0;
            if (i > 0 && !mbar_wait_warp(&full[st0], (it / AR_STAGES) & 1)) { ok = false; break; }
            if (two && !mbar_wait_warp(&full[st1], ((it + 1) / AR_STAGES) & 1)) { ok = false; break; }
            const int kt0 = tile_of[st0], kt1 = two ? tile_of[st1] : -1;
            const bool pre0 = ALONE && kt0 >= AR_PREFIX, pre1 = ALONE && kt1 >= AR_PREFIX;             // of a prefix: every row sees all of it
            const int kb0 = (ALONE ? kt0 & (AR_PREFIX - 1) : kt0) * TK + wk * 16, kb1 = (ALONE ? kt1 & (AR_PREFIX - 1) : kt1) * TK + wk * 16;     // first key of this warp's in either
            auto seen = [&](int kt, int kb, bool pre) { return kt >= 0 && (pre ? kb < u.key_lo : kb < any_hi && (kb + 16 > any_lo || kb < a.sinks)); };
            auto whole = [&](int kt, int kb, bool pre) { return kt >= 0 && (pre ? kb + 16 <= u.key_lo : kb + 16 <= all_hi && (kb >= all_lo || kb + 16 <= a.sinks)); };
            const bool in0 = seen(kt0, kb0, pre0), in1 = seen(kt1, kb1, pre1);
            if (in0 || in1) {
                const uint8_t* base[2] = {smem + st0 * AR_STAGE + wh * Cfg::HEAD, smem + st1 * AR_STAGE + wh * Cfg::HEAD};
                float s[4][4];                                                      // blocks of 8 keys, two of either tile
                #pragma unroll
                for (int nb = 0; nb < 4; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
                #pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t kf[4][4];
                    #pragma unroll
                    for (int nb = 0; nb < 4; ++nb) {
                        const int r = wk * 16 + (nb & 1) * 8 + (lane & 7), ch = x * 4 + (lane >> 3);      // row, 16-byte chunk of its 16
                        ldsm_x4(kf[nb][0], kf[nb][1], kf[nb][2], kf[nb][3], base[nb >> 1] + r * 128 + (ch >> 3) * Cfg::HALF + (((ch & 7) ^ (r & 7)) << 4));
                    }
                    #pragma unroll
                    for (int nb = 0; nb < 4; ++nb) mma_f16(s[nb], qf[2 * x][0], qf[2 * x][1], qf[2 * x][2], qf[2 * x][3], kf[nb][0], kf[nb][1]);
                    #pragma unroll
                    for (int nb = 0; nb < 4; ++nb) mma_f16(s[nb], qf[2 * x + 1][0], qf[2 * x + 1][1], qf[2 * x + 1][2], qf[2 * x + 1][3], kf[nb][2], kf[nb][3]);
                }
                // values of the first tile are asked for under the softmax, of the second under the first product
                const int vr = wk * 16 + (lane & 15);
                uint32_t vf[8][4];
                auto values = [&](int tile) {
                    #pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int ch = 2 * x + (lane >> 4);
                        ldsm_x4_t(vf[x][0], vf[x][1], vf[x][2], vf[x][3], base[tile] + AR_STAGE / 2 + vr * 128 + (ch >> 3) * Cfg::HALF + (((ch & 7) ^ (vr & 7)) << 4));
                    }
                };
                values(0);
                const bool clear = whole(kt0, kb0, pre0) && whole(kt1, kb1, pre1);              // every row sees every key of both
                uint32_t keep[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};      // values of keys that some row sees: pairs 2 t4, + 1 and 8 on
                float mx[2] = {-INFINITY, -INFINITY};
                #pragma unroll
                for (int nb = 0; nb < 4; ++nb)
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = __fmul_rn(s[nb][e], a.scale_log2);      // rounded here as in the maximum: not fused with the subtraction below
                        if (!clear) {
                            const int key = (nb < 2 ? kb0 : kb1) + (nb & 1) * 8 + 2 * t4 + (e & 1), h = e >> 1;
                            const bool in = nb < 2 ? in0 : in1, pre = nb < 2 ? pre0 : pre1;
                            if (!(in && (pre ? key < u.key_lo : key < hi[h] && (key >= lo[h] || key < a.sinks)))) v = -INFINITY;
                            if (!(in && (pre ? key < u.key_lo : key < any_hi && (key >= any_lo || key < a.sinks)))) keep[nb] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
                        }
                        s[nb][e] = v;
                        mx[e >> 1] = fmaxf(mx[e >> 1], v);
                    }
                float corr[2], ref[2];
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                    const float m_new = fmaxf(m_run[h], mx[h]);
                    corr[h] = m_new == -INFINITY ? 1.0f : ex2_approx(m_run[h] - m_new);
                    m_run[h] = m_new;
                    l_run[h] *= corr[h];
                    ref[h] = m_new == -INFINITY ? 0.f : m_new;       // a row that has seen nothing: exp2(-inf - 0) = 0
                }
                if (__any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f)) {
                    #pragma unroll
                    for (int d = 0; d < 16; ++d) { o_acc[d][0] *= corr[0]; o_acc[d][1] *= corr[0]; o_acc[d][2] *= corr[1]; o_acc[d][3] *= corr[1]; }
                }
                uint32_t pf[4][2];
                #pragma unroll
                for (int nb = 0; nb < 4; ++nb) {
                    const float e0 = ex2_approx(s[nb][0] - ref[0]), e1 = ex2_approx(s[nb][1] - ref[0]);
                    const float e2 = ex2_approx(s[nb][2] - ref[1]), e3 = ex2_approx(s[nb][3] - ref[1]);
                    l_run[0] += e0 + e1; l_run[1] += e2 + e3;
                    pf[nb][0] = pack_h2(e0, e1); pf[nb][1] = pack_h2(e2, e3);        // the one rounding of a weight, as the product takes it
                }
                #pragma unroll
                for (int tile = 0; tile < 2; ++tile) {
                    if (tile) values(1);
                    #pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        if (!clear) { vf[x][0] &= keep[2 * tile]; vf[x][1] &= keep[2 * tile + 1]; vf[x][2] &= keep[2 * tile]; vf[x][3] &= keep[2 * tile + 1]; }
                        mma_f16(o_acc[2 * x], pf[2 * tile][0], pf[2 * tile][1], pf[2 * tile + 1][0], pf[2 * tile + 1][1], vf[x][0], vf[x][1]);
                        mma_f16(o_acc[2 * x + 1], pf[2 * tile][0], pf[2 * tile][1], pf[2 * tile + 1][0], pf[2 * tile + 1][1], vf[x][2], vf[x][3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) { mbar_arrive(&empty[st0]); if (two) mbar_arrive(&empty[st1]); }
            it += two ? 2 : 1;
        }
        if (!ok) break;
        if (!u.whole) { const volatile ArUnit& v = units[n_unit % AR_UNITS]; u.c0 = v.c0; u.pieces = v.pieces; }

        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
        }
        auto place = [&](int r) -> size_t {              // (row, head) of the unit's row r
            const int qi = r / G;
            return (size_t)(u.row_base + qi) * a.nq + kvh * G + (r - qi * G);
        };
        auto part = [&](int k, int r) -> float* {        // partial sum of piece k
            return p.partial + (((size_t)(2 * (u.c0 + k) + (k == 0 ? 1 : 0)) * HW + wh) * AR_ROWS + r) * AR_MS;
        };
        if constexpr (KW == 1) {
            // ---- a warp has its head's rows: to the output, to where the prefix is added, or to the unit's partial sums
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = g + 8 * h;
                if (!valid[h]) continue;
                if (u.whole && u.group < 0) {
                    const float inv = l_run[h] > 0.f ? 1.0f / l_run[h] : 0.f;
                    uint32_t* to = reinterpret_cast<uint32_t*>(a.o + place(r) * 128) + t4;
                    #pragma unroll
                    for (int d = 0; d < 16; ++d) to[4 * d] = pack_h2(o_acc[d][2 * h] * inv, o_acc[d][2 * h + 1] * inv);
                } else {
                    float* to = u.whole ? p.rest + place(r) * AR_MS : p.partial + (((size_t)u.slot * HW + wh) * AR_ROWS + r) * AR_MS;
                    #pragma unroll
                    for (int d = 0; d < 16; ++d) *reinterpret_cast<float2*>(to + d * 8 + 2 * t4) = make_float2(o_acc[d][2 * h], o_acc[d][2 * h + 1]);
                    if (t4 == 0) *reinterpret_cast<float2*>(to + 128) = make_float2(m_run[h], l_run[h]);
                }
            }
            if (u.whole) continue;
            __threadfence();
            __syncwarp();
            int before = 0;
            if (lane == 0) {
                before = atomicAdd(p.counters + u.c0 * AR_WARPS + warp, 1);
                if (before == u.pieces - 1) p.counters[u.c0 * AR_WARPS + warp] = 0;
            }
            if (__shfl_sync(0xffffffffu, before, 0) != u.pieces - 1) continue;
            __threadfence();
            auto join = [&](auto rows_at_once, auto ahead) {
                constexpr int U = decltype(rows_at_once)::value;
                for (int r0 = 0; r0 < n_rows; r0 += U) {
                    SpanSum sums[U];
                    span_merge<decltype(ahead)::value>(sums, u.pieces, [&](int k, int i) -> const float* { return part(k, min(r0 + i, n_rows - 1)); },
                                                       [](int, int) { return true; }, lane);
                    #pragma unroll
                    for (int i = 0; i < U; ++i)
                        if (r0 + i < n_rows) span_put(a, p.rest, u.group, place(r0 + i), sums[i], lane);
                }
            };
            if (u.pieces <= 2) join(ArInt<8>(), ArInt<2>()); else join(ArInt<4>(), ArInt<4>());
        } else {
            // ---- the sums of the warps of a head: a common maximum, then one warp after the other adds to the buffer
            float* merge = reinterpret_cast<float*>(smem + Cfg::OFF_MERGE) + wh * AR_ROWS * AR_MS;
            #pragma unroll
            for (int h = 0; h < 2; ++h)
                if (t4 == 0) ml[warp * AR_ROWS + g + 8 * h] = make_float2(m_run[h], l_run[h]);
            if (!(ok = rendezvous())) break;
            float mm[2], ll[2];
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                mm[h] = -INFINITY; ll[h] = 0.f;
                #pragma unroll
                for (int w = 0; w < KW; ++w) mm[h] = fmaxf(mm[h], ml[(wh * KW + w) * AR_ROWS + g + 8 * h].x);
                #pragma unroll
                for (int w = 0; w < KW; ++w) {
                    const float2 x = ml[(wh * KW + w) * AR_ROWS + g + 8 * h];
                    ll[h] += x.x == -INFINITY ? 0.f : x.y * exp2f(x.x - mm[h]);
                }
                const float sc = m_run[h] == -INFINITY ? 0.f : exp2f(m_run[h] - mm[h]);
                #pragma unroll
                for (int d = 0; d < 16; ++d) { o_acc[d][2 * h] *= sc; o_acc[d][2 * h + 1] *= sc; }
            }
            for (int w = 0; w < KW && ok; ++w) {
                if (wk == w) {
                    #pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (valid[h]) {
                            float* row = merge + (g + 8 * h) * AR_MS;
                            #pragma unroll
                            for (int d = 0; d < 16; ++d) {
                                float2* at = reinterpret_cast<float2*>(row + d * 8 + 2 * t4);
                                float2 v = make_float2(o_acc[d][2 * h], o_acc[d][2 * h + 1]);
                                if (w > 0) { const float2 x = *at; v.x += x.x; v.y += x.y; }
                                *at = v;
                            }
                            if (w == 0 && t4 == 0) { row[128] = mm[h]; row[129] = ll[h]; }
                        }
                }
                ok = rendezvous();
            }
            if (!ok) break;
            // ---- a row per warp, four dims per lane
            constexpr int U = AR_ROWS / KW;              // a warp's rows: wk, wk + KW, ..
            bool finish = true;
            if (!u.whole) {
                for (int r = wk; r < n_rows; r += KW) {
                    float* to = p.partial + (((size_t)u.slot * HW + wh) * AR_ROWS + r) * AR_MS;
                    reinterpret_cast<float4*>(to)[lane] = reinterpret_cast<const float4*>(merge + r * AR_MS)[lane];
                    if (lane == 0) *reinterpret_cast<float2*>(to + 128) = *reinterpret_cast<const float2*>(merge + r * AR_MS + 128);
                }
                __threadfence();
                if (!(ok = rendezvous())) break;
                if (tid == 0) {
                    const int before = atomicAdd(p.counters + u.c0 * AR_WARPS, 1);
                    s_last = before == u.pieces - 1;
                    if (s_last) p.counters[u.c0 * AR_WARPS] = 0;
                }
                if (!(ok = rendezvous())) break;
                finish = s_last != 0;
                __threadfence();
            }
            if (finish) {
                #pragma unroll
                for (int i0 = 0; i0 < U; i0 += 4) {
                    SpanSum sums[4];
                    auto row = [&](int i) { return wk + KW * (i0 + i); };
                    if (u.whole) {
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float* at = merge + min(row(i), AR_ROWS - 1) * AR_MS;
                            if (row(i) < n_rows) sums[i] = {reinterpret_cast<const float4*>(at)[lane], at[128], at[129]};
                        }
                    } else
                        span_merge<4>(sums, u.pieces, [&](int k, int i) -> const float* { return part(k, min(row(i), n_rows - 1)); },
                                   [](int, int) { return true; }, lane);
                    #pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (row(i) < n_rows) span_put(a, p.rest, u.group, place(row(i)), sums[i], lane);
                }
            }
            if (!(ok = rendezvous())) break;            // the buffer is free again
        }
    }
    if (!p.first) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!ok && lane == 0) atomicExch(p.status, 3);
}

}  // namespace exl3
