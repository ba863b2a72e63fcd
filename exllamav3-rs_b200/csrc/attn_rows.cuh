// Attention over spans of the cache for sequences of few rows: at most 16 (query, head) rows per kv head, a decode row with its sibling
// heads or a few of them.
//
// Bound by HBM: every visible key and value is read once, and the two products are far below what mma.sync gives.  So the work is a
// stream: all sequences' key tiles of 64, head after head, stand in one line, and every CTA takes an equal part of it, whatever the
// lengths (148 SMs x 2 CTAs; the parts are found from the lengths by each CTA itself, so there is no list to build in front).  A
// producer warp runs ahead through a ring of three tiles and over the borders of sequences, so that the end of one costs no loads.
// A sequence and head whose tiles fall to several CTAs goes through partial sums, which the CTA that arrives last adds up in the order of
// the tiles: results do not depend on who that is.
//
// Four warps take 16 keys of a tile each with a softmax state of their own, and meet at the end of a unit.  Keys of a tile that no row sees
// are not loaded where they fill a group of 16, and masked in both products where not (a masked key's value may be NaN).
#pragma once
#include <cuda.h>
#include "attn_span.cuh"
#include "attn_paged.cuh"
#include "async_copy.cuh"

namespace exl3 {

constexpr int AR_TK = 64, AR_ROWS = 16, AR_STAGES = 3, AR_WARPS = 4;
constexpr int AR_THREADS = (AR_WARPS + 1) * 32;
constexpr int AR_HALF = AR_TK * 128;                    // bytes of one 64-dim half of a tile: rows of 128 bytes, 128-byte swizzle
constexpr int AR_STAGE = 4 * AR_HALF;                   // K and V
constexpr int AR_MS = SPAN_PART;
constexpr int AR_MAX_BSZ = 1024;                        // sequences of a launch: their tile counts are summed in shared memory
constexpr int AR_UNITS = AR_STAGES + 1;                 // unit descriptors: the producer is at most AR_STAGES tiles, so units, ahead

struct ArUnit { int b, kvh, row_base, ql, cached, key_lo, group, whole, slot, c0, pieces, tiles; };

struct ArSmem {
    static constexpr int OFF_MERGE = AR_STAGES * AR_STAGE;
    static constexpr int OFF_ML = OFF_MERGE + AR_ROWS * AR_MS * 4;
    static constexpr int OFF_SUM = OFF_ML + AR_WARPS * AR_ROWS * 8;
    static constexpr int OFF_UNIT = OFF_SUM + (AR_MAX_BSZ + 4) * 4;
    static constexpr int OFF_BAR = OFF_UNIT + AR_UNITS * (int)sizeof(ArUnit);
    // full[stages], empty[stages], meet; then the tile of every stage
    static constexpr int OFF_TILE = OFF_BAR + (2 * AR_STAGES + 1) * 8;
    static constexpr int BYTES = OFF_TILE + AR_STAGES * 4 + 16 + 1024;
};
static_assert(2 * (ArSmem::BYTES + 1024) <= EXL3_SM_SMEM, "two CTAs per SM");

struct ArMaps { CUtensorMap k, v, k16, v16; };          // boxes of 64 tokens x 2 halves, and of 16 tokens x 1 half

struct ArParams {
    SpanArgs a;
    int b0, bsz;                                        // sequences of this launch
    int min_share;                                      // tiles that a CTA takes at least
    float* partial;                                     // [2 * CTAs][16][AR_MS]
    int* counters;                                      // [CTAs], zero between calls
    int* status;
    float* rest;                                        // [rows][nq][AR_MS] partial sums of sequences that a prefix is added to
    int first;                                          // nothing of this call is in front of the launch
};

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4, uint64_t* bar)
{
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar)) : "memory");
}

__global__ void __launch_bounds__(AR_THREADS, 2) attn_rows_kernel(const __grid_constant__ ArMaps maps, const ArParams p, int early)
{
    if (p.first) pdl_enter_first(early);
    else asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint8_t smem_unaligned[];
    uint8_t* smem = smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u);
    float* merge = reinterpret_cast<float*>(smem + ArSmem::OFF_MERGE);
    float2* ml = reinterpret_cast<float2*>(smem + ArSmem::OFF_ML);                  // [warp][row]
    int* sum = reinterpret_cast<int*>(smem + ArSmem::OFF_SUM);                      // [bsz + 1] first tile of every sequence, per head
    ArUnit* units = reinterpret_cast<ArUnit*>(smem + ArSmem::OFF_UNIT);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + ArSmem::OFF_BAR);
    uint64_t* empty = full + AR_STAGES;
    uint64_t* meet = empty + AR_STAGES;
    int* tile_of = reinterpret_cast<int*>(smem + ArSmem::OFF_TILE);                 // key tile in a stage, -1: none of its keys exist
    __shared__ int s_last;

    const SpanArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.nq / a.nkv;
    if (tid == 0) {
        for (int i = 0; i < AR_STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], AR_WARPS); }
        mbar_init(meet, AR_WARPS);
        mbar_fence_init();
    }
    // a sequence's tiles, at least one if it has rows of this kernel (their output is written)
    auto key_lo_of = [&](int b, int cached, int* group) -> int {
        const SpanGroup g = span_group(a, b, cached);
        *group = g.g;
        return g.len;
    };
    auto tiles_of = [&](int b) -> int {
        const SpanSeq s = span_seq(a, b);
        if (s.ql == 0 || s.ql * G > AR_ROWS) return 0;
        int group;
        const SpanTiles t = span_tiles<AR_TK>(a, s.cached, s.cached + s.ql - 1, key_lo_of(b, s.cached, &group));
        return max(t.sink + t.near, 1);
    };
    for (int b = tid; b < p.bsz; b += AR_THREADS) sum[b] = tiles_of(p.b0 + b);
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
    // this CTA's part [f0, f1) of the line of all tiles: sequence, head, tile
    const long long F = (long long)sum[p.bsz] * a.nkv;
    const long long want = (F + p.min_share - 1) / p.min_share;
    const int C = (int)min((long long)gridDim.x, max(want, 1LL));
    const int c = blockIdx.x;
    const long long f0 = c < C ? c * F / C : F, f1 = c < C ? (c + 1) * F / C : F;
    if (f0 >= f1) {
        if (!p.first) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    auto cta_of = [&](long long f) -> int { return (int)(((f + 1) * C - 1) / F); };

    if (warp == AR_WARPS) {
        // ===== producer: the whole warp walks, lane 0 issues; lane i holds the block table's entry page0 + i
        int it = 0, n_unit = 0;
        long long f = f0;
        int b = 0;
        {
            const int per_head = (int)(f0 / a.nkv);     // last sequence whose first tile is not behind f0: sum[b] * nkv <= f0
            int lo = 0, hi = p.bsz;
            while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (sum[mid] <= per_head) lo = mid; else hi = mid; }
            b = lo;
        }
        bool ok = true;
        SpanSeq s = {0, 0, 0};
        SpanTiles t = {};
        int key_lo = 0, group = -1, have = -1, page0 = 0, entry = 0;
        while (f < f1 && ok) {
            while ((long long)sum[b + 1] * a.nkv <= f) ++b;
            const int n = sum[b + 1] - sum[b];
            const int in = (int)(f - (long long)sum[b] * a.nkv), kvh = in / n, from = in - kvh * n;
            const int upto = (int)min((long long)n, from + (f1 - f));
            const int gb = p.b0 + b;
            const int32_t* bt = a.block_table + (size_t)gb * a.pps;
            if (have != b) {
                s = span_seq(a, gb);
                key_lo = key_lo_of(gb, s.cached, &group);
                t = span_tiles<AR_TK>(a, s.cached, s.cached + s.ql - 1, key_lo);
                page0 = -64; have = b;
            }
            const long long u0 = f - from;
            for (int i = from; i < upto; ++i, ++it) {
                const int stage = it % AR_STAGES;
                const int kt = t.sink + t.near == 0 ? -1 : i < t.sink ? i : t.first + (i - t.sink);
                int page = -1;
                if (kt >= 0) {
                    const int pg = kt / (EXL3_PAGE / AR_TK);
                    if (pg < page0 || pg >= page0 + 32) { page0 = pg; entry = pg + lane < a.pps ? bt[pg + lane] : -1; }
                    page = __shfl_sync(0xffffffffu, entry, pg - page0);
                    if (page >= a.pages) page = -1;
                }
                if (it >= AR_STAGES && !mbar_wait_sleep_warp(&empty[stage], ((it / AR_STAGES) - 1) & 1)) { ok = false; break; }
                if (lane == 0) {
                    if (i == from) {
                        ArUnit& u = units[n_unit % AR_UNITS];
                        u.b = gb; u.kvh = kvh; u.row_base = s.row_base; u.ql = s.ql; u.cached = s.cached; u.key_lo = key_lo; u.group = group;
                        u.whole = from == 0 && upto == n;
                        u.slot = 2 * c + (from == 0 ? 1 : 0);
                        u.c0 = cta_of(u0); u.pieces = cta_of(u0 + n - 1) - u.c0 + 1; u.tiles = upto - from;
                    }
                    tile_of[stage] = page < 0 ? -1 : kt;
                    if (page < 0) mbar_arrive(&full[stage]);
                    else {
                        // groups of 16 keys with one that some row sees
                        const int k0 = kt * AR_TK, tok = k0 & (EXL3_PAGE - 1);
                        const int hi = min(AR_TK, (i < t.sink ? min(a.sinks, t.end) : t.end) - k0);
                        const int lo = i < t.sink || a.sinks > k0 ? 0 : max(0, t.lo - k0);
                        const int g0 = lo >> 4, g1 = (hi + 15) >> 4;
                        uint8_t* st = smem + stage * AR_STAGE;
                        if (g1 - g0 == 4) {
                            mbar_expect_tx(&full[stage], AR_STAGE);
                            tma_load_5d(st, &maps.k, 0, tok, 0, kvh, page, &full[stage]);
                            tma_load_5d(st + 2 * AR_HALF, &maps.v, 0, tok, 0, kvh, page, &full[stage]);
                        } else {
                            mbar_expect_tx(&full[stage], (g1 - g0) * (AR_STAGE / 4));
                            for (int g = g0; g < g1; ++g)
                                for (int h = 0; h < 2; ++h) {
                                    tma_load_5d(st + h * AR_HALF + g * 2048, &maps.k16, 0, tok + 16 * g, h, kvh, page, &full[stage]);
                                    tma_load_5d(st + (2 + h) * AR_HALF + g * 2048, &maps.v16, 0, tok + 16 * g, h, kvh, page, &full[stage]);
                                }
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

    // ===== four warps, 16 keys of every tile each
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
        const ArUnit u = units[n_unit % AR_UNITS];
        f += u.tiles;
        const int n_rows = u.ql * G;
        int lo[2], hi[2];
        bool valid[2];
        uint32_t qf[8][4];
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = g + 8 * h, qi = row / G, pos = u.cached + qi;
            valid[h] = row < n_rows;
            hi[h] = min(max(pos + 1, 0), a.pps * EXL3_PAGE);
            lo[h] = max(u.key_lo, a.window > pos ? 0 : pos - a.window + 1);
            const half* qp = a.q + ((size_t)(u.row_base + qi) * a.nq + u.kvh * G + (row - qi * G)) * 128;
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
        for (int i = 0; i < u.tiles; ++i, ++it) {
            const int stage = it % AR_STAGES;
            if (i > 0 && !mbar_wait_warp(&full[stage], (it / AR_STAGES) & 1)) { ok = false; break; }
            const int kt = tile_of[stage];
            const int kb = kt * AR_TK + warp * 16;                                   // first key of this warp's
            if (kt >= 0 && kb < any_hi && (kb + 16 > any_lo || kb < a.sinks)) {
                const uint8_t* ks_ = smem + stage * AR_STAGE;
                const uint8_t* vs_ = ks_ + 2 * AR_HALF;
                float s[2][4];
                #pragma unroll
                for (int nb = 0; nb < 2; ++nb) {
                    s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
                    const int r = warp * 16 + nb * 8 + (lane & 7);
                    const uint8_t* krow = ks_ + r * 128;
                    #pragma unroll
                    for (int ks = 0; ks < 8; ks += 2) {
                        const int ch = ks * 2 + (lane >> 3);                         // 16-byte chunk of the row's 16
                        uint32_t b0, b1, b2, b3;
                        ldsm_x4(b0, b1, b2, b3, krow + (ch >> 3) * AR_HALF + (((ch & 7) ^ (r & 7)) << 4));
                        mma_f16(s[nb], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b0, b1);
                        mma_f16(s[nb], qf[ks + 1][0], qf[ks + 1][1], qf[ks + 1][2], qf[ks + 1][3], b2, b3);
                    }
                }
                const bool clear = kb + 16 <= all_hi && (kb >= all_lo || kb + 16 <= a.sinks);      // every row sees every key
                uint32_t keep[2] = {0xffffffffu, 0xffffffffu};                       // values of keys that exist for some row: pairs 2 t4, + 1 and 8 on
                float mx[2] = {-INFINITY, -INFINITY};
                #pragma unroll
                for (int nb = 0; nb < 2; ++nb)
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = s[nb][e] * a.scale_log2;
                        if (!clear) {
                            const int key = kb + nb * 8 + 2 * t4 + (e & 1), h = e >> 1;
                            if (!(key < hi[h] && (key >= lo[h] || key < a.sinks))) v = -INFINITY;
                            if (!(key < any_hi && (key >= any_lo || key < a.sinks))) keep[nb] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
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
                    corr[h] = m_new == -INFINITY ? 1.0f : exp2f(m_run[h] - m_new);
                    m_run[h] = m_new;
                    l_run[h] *= corr[h];
                    ref[h] = m_new == -INFINITY ? 0.f : m_new;       // a row that has seen nothing: exp2(-inf - 0) = 0
                }
                if (__any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f)) {
                    #pragma unroll
                    for (int d = 0; d < 16; ++d) { o_acc[d][0] *= corr[0]; o_acc[d][1] *= corr[0]; o_acc[d][2] *= corr[1]; o_acc[d][3] *= corr[1]; }
                }
                uint32_t pf[2][2];
                #pragma unroll
                for (int nb = 0; nb < 2; ++nb) {
                    const float e0 = exp2f(s[nb][0] - ref[0]), e1 = exp2f(s[nb][1] - ref[0]);
                    const float e2 = exp2f(s[nb][2] - ref[1]), e3 = exp2f(s[nb][3] - ref[1]);
                    l_run[0] += e0 + e1; l_run[1] += e2 + e3;
                    pf[nb][0] = pack_h2(e0, e1); pf[nb][1] = pack_h2(e2, e3);        // the one rounding of a weight, as the product takes it
                }
                const int vr = warp * 16 + (lane & 15);
                const uint8_t* vrow = vs_ + vr * 128;
                #pragma unroll
                for (int db = 0; db < 16; db += 2) {
                    const int ch = db + (lane >> 4);
                    uint32_t b0, b1, b2, b3;
                    ldsm_x4_t(b0, b1, b2, b3, vrow + (ch >> 3) * AR_HALF + (((ch & 7) ^ (vr & 7)) << 4));
                    if (!clear) { b0 &= keep[0]; b1 &= keep[1]; b2 &= keep[0]; b3 &= keep[1]; }
                    mma_f16(o_acc[db], pf[0][0], pf[0][1], pf[1][0], pf[1][1], b0, b1);
                    mma_f16(o_acc[db + 1], pf[0][0], pf[0][1], pf[1][0], pf[1][1], b2, b3);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
        }
        if (!ok) break;

        // ---- the four warps' sums: a common maximum, then one warp after the other adds to the buffer
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
            if (t4 == 0) ml[warp * AR_ROWS + g + 8 * h] = make_float2(m_run[h], l_run[h]);
        }
        if (!(ok = rendezvous())) break;
        float mm[2], ll[2];
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            mm[h] = -INFINITY; ll[h] = 0.f;
            #pragma unroll
            for (int w = 0; w < AR_WARPS; ++w) mm[h] = fmaxf(mm[h], ml[w * AR_ROWS + g + 8 * h].x);
            #pragma unroll
            for (int w = 0; w < AR_WARPS; ++w) {
                const float2 x = ml[w * AR_ROWS + g + 8 * h];
                ll[h] += x.x == -INFINITY ? 0.f : x.y * exp2f(x.x - mm[h]);
            }
            const float sc = m_run[h] == -INFINITY ? 0.f : exp2f(m_run[h] - mm[h]);
            #pragma unroll
            for (int d = 0; d < 16; ++d) { o_acc[d][2 * h] *= sc; o_acc[d][2 * h + 1] *= sc; }
        }
        for (int w = 0; w < AR_WARPS && ok; ++w) {
            if (warp == w) {
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
        bool finish = u.whole != 0;
        if (!u.whole) {
            float* part = p.partial + (size_t)u.slot * AR_ROWS * AR_MS;
            for (int r = warp; r < n_rows; r += AR_WARPS) {
                reinterpret_cast<float4*>(part + r * AR_MS)[lane] = reinterpret_cast<const float4*>(merge + r * AR_MS)[lane];
                if (lane == 0) *reinterpret_cast<float2*>(part + r * AR_MS + 128) = *reinterpret_cast<const float2*>(merge + r * AR_MS + 128);
            }
            __threadfence();
            if (!(ok = rendezvous())) break;
            if (tid == 0) {
                const int before = atomicAdd(p.counters + u.c0, 1);
                s_last = before == u.pieces - 1;
                if (s_last) p.counters[u.c0] = 0;
            }
            if (!(ok = rendezvous())) break;
            finish = s_last != 0;
            __threadfence();
        }
        if (finish) {
            constexpr int U = AR_ROWS / AR_WARPS;           // a warp's rows: warp, warp + 4, ..
            bool on[U];
            SpanSum sum[U];
            size_t at[U];
            #pragma unroll
            for (int i = 0; i < U; ++i) {
                on[i] = warp + AR_WARPS * i < n_rows;
                const int r = on[i] ? warp + AR_WARPS * i : 0, qi = r / G;       // (a row that is not there stands for the first one)
                at[i] = (size_t)(u.row_base + qi) * a.nq + u.kvh * G + (r - qi * G);
            }
            if (u.whole) {
                #pragma unroll
                for (int i = 0; i < U; ++i) {
                    const float* row = merge + (warp + AR_WARPS * i) * AR_MS;
                    if (on[i]) sum[i] = {reinterpret_cast<const float4*>(row)[lane], row[128], row[129]};
                }
            } else
                span_merge(sum, u.pieces, [&](int k, int i) -> const float* {
                    return p.partial + ((size_t)(2 * (u.c0 + k) + (k == 0 ? 1 : 0)) * AR_ROWS + (on[i] ? warp + AR_WARPS * i : 0)) * AR_MS; },
                    [](int, int) { return true; }, lane);
            #pragma unroll
            for (int i = 0; i < U; ++i) {
                if (!on[i]) continue;
                if (u.group < 0) reinterpret_cast<uint2*>(a.o)[at[i] * 32 + lane] = span_result(sum[i]);
                else {                                          // span_join_kernel adds the prefix
                    reinterpret_cast<float4*>(p.rest + at[i] * AR_MS)[lane] = sum[i].acc;
                    if (lane == 0) *reinterpret_cast<float2*>(p.rest + at[i] * AR_MS + 128) = make_float2(sum[i].top, sum[i].l);
                }
            }
        }
        if (!(ok = rendezvous())) break;                // the buffer is free again
    }
    if (!p.first) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!ok && lane == 0) atomicExch(p.status, 3);
}

}  // namespace exl3
