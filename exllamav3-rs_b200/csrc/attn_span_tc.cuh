// Attention over spans of the cache on tcgen05: sequences with more than 16 (query, head) rows per kv head, and the shared prefixes, whose
// rows are those of all sequences of a group.
//
// An item is NB blocks of 128 packed rows of one kv head and a run of key tiles of 128.  S = Q K^T (128 x 128) and O += P V are 128-column
// accumulators in tensor memory per block, P goes back over the first half of S as packed fp16 and is the A operand of the second
// product.  One softmax thread owns a row, so maxima and sums need no exchange.
//
// What bounds it: per tile and row block 776 + 512 cycles of the tensor core (128 x 128 x 16 with A in shared memory takes 97 cycles, in
// tensor memory 64), 1024 of the special-function unit (16 exponentials per clock and SM) and 64 KB of keys and values out of L2, in a
// chain of scores, softmax, product that a block cannot overlap with itself.  So an SM holds two blocks, whose softmax runs under the
// other's products: NB = 2, one CTA whose blocks share every tile, where sequences have the rows (with two CTAs that read tiles of their own
// 4 x 2048 rows took 794 us: 64 KB per 2500 cycles and SM is what L2 gives); NB = 1, two CTAs of one block, where they do not, so that
// the start and end of short items overlap.
//
// Items are found by every CTA from the lengths themselves (warp 0, entries over lanes), which costs about a microsecond and saves a launch
// in front.  A run of tiles is cut into as many splits as fill the GPU, by the same rule in every CTA.
#pragma once
#include "attn_rows.cuh"
#include "attn_tc_ops.cuh"

namespace exl3 {

constexpr int AS_BLOCK = 128;                            // rows of a block: the lanes of tensor memory
constexpr int AS_TILE = AS_TK * 256;                    // bytes of a tile of K, V or Q: two 64-dim halves of 16 KB
constexpr int AS_MAX_SPLITS = 32;
constexpr int AS_ITEM_COST = 4;                         // start and end of an item, in tiles

template <int NB>
struct AsCfg {
    static constexpr int ROWS = AS_BLOCK * NB, SW = 4 * NB, THREADS = (SW + 2) * 32;       // softmax warps, TMA producer, MMA issuer
    static constexpr int SLOTS = NB == 1 ? 2 : 5;                                          // ring of tiles: K0 V0 K1 V1 ...
    static constexpr int OFF_Q = 0, OFF_KV = NB * AS_TILE, OFF_BAR = OFF_KV + SLOTS * AS_TILE;
    static constexpr int NBARS = 4 * NB + 2 * SLOTS + 1;                                   // q_full, s_full, p_half, p_full per block; full, empty per slot; o_full
    static constexpr int SMEM = OFF_BAR + NBARS * 8 + 16 + 1024;
    static constexpr int CTAS = NB == 1 ? 2 : 1, TMEM = 256 * NB;
    static_assert(ROWS * SPAN_PART * 4 <= (NB + SLOTS) * AS_TILE, "partial sums are staged over the tiles");
    static_assert(CTAS * (SMEM + 1024) <= EXL3_SM_SMEM, "CTAs of an SM");
};

struct AsParams {
    SpanArgs a;
    float* partial;                                     // [splits][rows][nq][SPAN_PART]
    int* chunk;                                         // key tiles per split, for the kernels behind
    int* status;
    int prefixes;                                       // 1: the groups' prefixes, 0: the sequences' own spans
    int max_splits, max_items, slots;
    int first;                                          // nothing of this call is in front of the launch
};
struct AsJoin {                                         // what the kernels behind find of both
    SpanArgs a;
    const float* prefix; const int* prefix_chunk;
    const float* own; const int* own_chunk;
    int own_rows;                                       // rows of an item of the sequences' own spans
};

// A run of rows over one run of keys, before it is cut into items
struct AsEntry { int tab, row_base, n_rows, ql, cached, key_lo, tiles; };

__device__ __forceinline__ int as_blocks(int packed, int rows) { return (packed + rows - 1) / rows; }
// tiles of a sequence's last row block, which has as many as any other but for alignment
__device__ __forceinline__ int as_own_tiles(const SpanArgs& a, const SpanSeq& s, int key_lo, int G, int rows)
{
    const int i_first = (as_blocks(s.ql * G, rows) - 1) * rows / G;
    const SpanTiles t = span_tiles<AS_TK>(a, s.cached + i_first, s.cached + s.ql - 1, key_lo);
    return t.sink + t.near;
}
__device__ __forceinline__ AsEntry as_entry(const AsParams& p, int e, int G, int rows)
{
    const SpanArgs& a = p.a;
    AsEntry r = {0, 0, 0, 0, 0, 0, 0};
    if (p.prefixes) {
        const int first = max(a.group_start[e], 0), last = min(a.group_start[e + 1], a.bsz);
        const int len = min(a.prefix_lens[e], a.pps * EXL3_PAGE);
        if (first >= last || len <= 0) return r;
        const int r0 = max(a.cu_q ? a.cu_q[first] : first * a.q_len, 0), r1 = min(a.cu_q ? a.cu_q[last] : last * a.q_len, a.rows);
        if (r0 >= r1) return r;
        r.tab = first; r.row_base = r0; r.ql = r1 - r0; r.cached = len; r.tiles = (len + AS_TK - 1) / AS_TK;
    } else {
        const SpanSeq s = span_seq(a, e);
        if (s.ql * G <= AR_ROWS) return r;
        r.tab = e; r.row_base = s.row_base; r.ql = s.ql; r.cached = s.cached;
        r.key_lo = span_group(a, e, s.cached).len;
        r.tiles = as_own_tiles(a, s, r.key_lo, G, rows);
    }
    r.n_rows = r.ql * G;
    return r;
}

struct AsItem { AsEntry e; int rb, split, splits, kvh; };

// The item of this CTA (warp-uniform, all lanes); false: there is none.  chunk: tiles per split, as all CTAs find it.
__device__ __forceinline__ bool as_item(const AsParams& p, int G, int rows, int lane, AsItem& it, int& chunk)
{
    const int nkv = p.a.nkv, n = p.prefixes ? p.a.n_groups : p.a.bsz;
    AsEntry e = {};
    if (lane < n) e = as_entry(p, lane, G, rows);       // of the first 32 entries, which are often all
    auto entry = [&](int e0) { if (n > 32) { e = {}; if (e0 + lane < n) e = as_entry(p, e0 + lane, G, rows); } };
    int most = 1;
    for (int e0 = 0; e0 < n; e0 += 32) { entry(e0); most = max(most, e.tiles); }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    // lane i weighs i + 1 splits of the longest run: waves of items times what an item takes
    const int mine = (most + lane) / (lane + 1);
    if (p.max_splits > 1) {
        long long items = 0;
        for (int e0 = 0; e0 < n; e0 += 32) {
            entry(e0);
            const int units = as_blocks(e.n_rows, rows) * nkv;
            unsigned live = __ballot_sync(0xffffffffu, units > 0);
            while (live) {
                const int j = __ffs(live) - 1;
                live &= live - 1;
                items += (long long)__shfl_sync(0xffffffffu, units, j) * as_splits(__shfl_sync(0xffffffffu, e.tiles, j), mine);
            }
        }
        long long cost = (items + p.slots - 1) / p.slots * (mine + AS_ITEM_COST);
        if (lane > 0 && (lane >= p.max_splits || items > p.max_items)) cost = 1LL << 60;
        int best = lane;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const long long c2 = __shfl_xor_sync(0xffffffffu, cost, o);
            const int b2 = __shfl_xor_sync(0xffffffffu, best, o);
            if (c2 < cost || (c2 == cost && b2 < best)) { cost = c2; best = b2; }
        }
        chunk = __shfl_sync(0xffffffffu, mine, best);
    } else chunk = most;
    int before = 0;
    for (int e0 = 0; e0 < n; e0 += 32) {
        entry(e0);
        const int rb = as_blocks(e.n_rows, rows), sp = as_splits(e.tiles, chunk), own = rb * nkv * sp;
        int v = own;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += u; }
        const int at = (int)blockIdx.x - before;
        const unsigned behind = __ballot_sync(0xffffffffu, v > at);
        if (behind) {
            const int j = __ffs(behind) - 1;
            const int in = at - __shfl_sync(0xffffffffu, v - own, j), n_rb = __shfl_sync(0xffffffffu, rb, j);
            it.splits = __shfl_sync(0xffffffffu, sp, j);
            it.e.tab = __shfl_sync(0xffffffffu, e.tab, j); it.e.row_base = __shfl_sync(0xffffffffu, e.row_base, j);
            it.e.n_rows = __shfl_sync(0xffffffffu, e.n_rows, j); it.e.ql = __shfl_sync(0xffffffffu, e.ql, j);
            it.e.cached = __shfl_sync(0xffffffffu, e.cached, j); it.e.key_lo = __shfl_sync(0xffffffffu, e.key_lo, j);
            it.e.tiles = __shfl_sync(0xffffffffu, e.tiles, j);
            // row blocks of a head and run are neighbours, which read the same keys; the last, the longest where it is causal, first
            it.rb = n_rb - 1 - in % n_rb; it.split = in / n_rb % it.splits; it.kvh = in / n_rb / it.splits;
            return true;
        }
        before += __shfl_sync(0xffffffffu, v, 31);
    }
    return false;
}

// two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    uint64_t x, y, z, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    float2 o;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
    return o;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    uint64_t x, y, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    float2 o;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
    return o;
}

template <int NB>
__global__ void __launch_bounds__(AsCfg<NB>::THREADS, AsCfg<NB>::CTAS) attn_span_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                                         const __grid_constant__ CUtensorMap vmap,
                                                                                         const AsParams p, int early)
{
    using Cfg = AsCfg<NB>;
    constexpr int SW = Cfg::SW, SLOTS = Cfg::SLOTS;
    (void)early;
    if (p.first) pdl_wait();
    extern __shared__ uint8_t smem_unaligned[];
    uint8_t* smem = smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
    uint64_t *q_full = bars, *s_full = q_full + NB, *p_half = s_full + NB, *p_full = p_half + NB, *kv_full = p_full + NB, *kv_empty = kv_full + SLOTS,
             *o_full = kv_empty + SLOTS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NBARS);
    __shared__ AsItem s_item;
    __shared__ int s_have, s_failed;

    const SpanArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.nq / a.nkv;
    if (warp == 0) {
        AsItem it;
        int chunk;
        const bool have = as_item(p, G, Cfg::ROWS, lane, it, chunk);
        if (lane == 0) {
            s_have = have; s_item = it; s_failed = 0;
            if (blockIdx.x == 0) *p.chunk = chunk;
        }
    }
    if (tid == 32) {
        for (int i = 0; i < NB; ++i) { mbar_init(&q_full[i], 4); mbar_init(&s_full[i], 1); mbar_init(&p_half[i], 4); mbar_init(&p_full[i], 4); }
        for (int i = 0; i < SLOTS; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
        mbar_init(o_full, 1);
        mbar_fence_init();
    }
    __syncthreads();
    if (!s_have) {
        if (!p.first) pdl_wait();
        return;
    }
    if (warp == SW + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Cfg::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    const AsEntry e = s_item.e;
    const int kvh = s_item.kvh, r0 = s_item.rb * Cfg::ROWS, n_valid = min(Cfg::ROWS, e.n_rows - r0), n_blocks = NB == 1 || n_valid <= AS_BLOCK ? 1 : 2;
    const int table_end = a.pps * EXL3_PAGE;
    const bool prefix = p.prefixes != 0;
    // the item's key tiles, and this split's part [t0, t1) of them
    SpanTiles t;
    int all_lo, all_hi, sinks;                              // what every row of the item sees
    if (prefix) {
        t.sink = 0; t.first = 0; t.near = e.tiles; t.lo = 0; t.end = e.cached;
        all_lo = 0; all_hi = e.cached; sinks = 0;
    } else {
        const int p_first = e.cached + r0 / G, p_last = e.cached + (r0 + n_valid - 1) / G;
        t = span_tiles<AS_TK>(a, p_first, p_last, e.key_lo);
        all_hi = min(max(p_first + 1, 0), table_end);
        all_lo = max(e.key_lo, a.window > p_last ? 0 : p_last - a.window + 1);
        sinks = a.sinks;
    }
    const int total = t.sink + t.near, t0 = (int)((long long)total * s_item.split / s_item.splits), t1 = (int)((long long)total * (s_item.split + 1) / s_item.splits);
    const int n_tiles = t1 - t0;
    auto key_tile = [&](int j) -> int { const int i = t0 + j; return i < t.sink ? i : t.first + (i - t.sink); };
    const int32_t* bt = a.block_table + (size_t)e.tab * a.pps;
    auto page_of = [&](int j) -> int { const int pg = bt[key_tile(j) >> 1]; return pg >= 0 && pg < a.pages ? pg : -1; };

    if (warp < SW && warp < 4 * n_blocks) {
        // a warp's 32 Q rows -> shared memory, K-major, 128-byte swizzle: half a warp per row
        const int c = lane & 15;
        uint8_t* qs = smem + Cfg::OFF_Q + (warp >> 2) * AS_TILE + (c >> 3) * (AS_TILE / 2);
        uint4 x[16];
        #pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = warp * 32 + 2 * i + (lane >> 4), pr = r0 + r, qi = pr / G;
            x[i] = make_uint4(0, 0, 0, 0);
            if (r < n_valid) x[i] = __ldg(reinterpret_cast<const uint4*>(a.q + ((size_t)(e.row_base + qi) * a.nq + kvh * G + (pr - qi * G)) * 128) + c);
        }
        #pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = (warp & 3) * 32 + 2 * i + (lane >> 4);
            *reinterpret_cast<uint4*>(qs + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = x[i];
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[warp >> 2]);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // kernels behind may be set up from here on (in front of the allocation they could take the tensor memory and wait for this one)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    bool failed = false;

    if (warp == SW) {
        // ===== producer
        if (lane == 0 && n_tiles > 0) {
            int page = page_of(0), it = 0;
            bool ok = true;
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int tok = (key_tile(j) * AS_TK) & (EXL3_PAGE - 1);
                const int pg = page < 0 ? a.pages : page;   // outside the pool: zeros, which the softmax threads mask
                if (j + 1 < n_tiles) page = page_of(j + 1);
                #pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int slot = it % SLOTS;
                    if (it >= SLOTS && !mbar_wait_sleep(&kv_empty[slot], ((it / SLOTS) - 1) & 1)) { ok = false; break; }
                    mbar_expect_tx(&kv_full[slot], AS_TILE);
                    tma_load_5d(smem + Cfg::OFF_KV + slot * AS_TILE, v ? &vmap : &kmap, 0, tok, 0, kvh, pg, &kv_full[slot]);
                    ++it;
                }
            }
            failed = !ok;
            // not out before every copy has landed, whatever became of those who take them
            for (int i = max(0, it - SLOTS); i < it; ++i) mbar_wait_sleep(&kv_full[i % SLOTS], (i / SLOTS) & 1);
        }
    } else if (warp == SW + 1) {
        // ===== MMA issuer: warp-uniform values, one elected lane
        if (n_tiles > 0) {
            const bool leader = elect_one();
            constexpr uint32_t HI = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);     // SBO, version 1, SWIZZLE_128B
            constexpr uint32_t LBO_K = 1u << 16, LBO_V = (uint32_t)((AS_TILE / 2) >> 4) << 16;
            auto mk = [](uint32_t lo, uint32_t hi) { return ((uint64_t)hi << 32) | lo; };
            const uint32_t q_lo = (smem_u32(smem + Cfg::OFF_Q) >> 4) | LBO_K, kv_lo = smem_u32(smem + Cfg::OFF_KV) >> 4;
            // S of a block from the K tile that is ring item 2 j
            auto scores = [&](int b, int j) -> bool {
                const int slot = (2 * j) % SLOTS;
                if (b == 0 && !mbar_wait_sleep_warp(&kv_full[slot], (2 * j / SLOTS) & 1)) return false;
                tc_fence_after();
                if (leader) {
                    const uint32_t qb = q_lo + b * (AS_TILE >> 4), kb = (kv_lo + slot * (AS_TILE >> 4)) | LBO_K;
                    #pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t off = ((kk >> 2) * (AS_TILE / 2) + (kk & 3) * 32) >> 4;
                        tc_mma_f16(tmem + b * 256, mk(qb + off, HI), mk(kb + off, HI), ATC_IDESC_S, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(&s_full[b]);
                    if (b == n_blocks - 1) tc_commit(&kv_empty[slot]);
                }
                __syncwarp();
                return true;
            };
            for (int b = 0; b < n_blocks && !failed; ++b)
                if (!mbar_wait_sleep_warp(&q_full[b], 0) || !scores(b, 0)) failed = true;
            for (int j = 0; j < n_tiles && !failed; ++j) {
                const int slot = (2 * j + 1) % SLOTS;
                for (int b = 0; b < n_blocks && !failed; ++b) {
                    if (b == 0 && !mbar_wait_sleep_warp(&kv_full[slot], ((2 * j + 1) / SLOTS) & 1)) { failed = true; break; }
                    const uint32_t vb = (kv_lo + slot * (AS_TILE >> 4)) | LBO_V, tb = tmem + b * 256;
                    #pragma unroll
                    for (int half_ = 0; half_ < 2 && !failed; ++half_) {
                        if (!mbar_wait_warp(half_ ? &p_full[b] : &p_half[b], j & 1)) { failed = true; break; }
                        tc_fence_after();
                        if (leader) {
                            #pragma unroll
                            for (int kk = 4 * half_; kk < 4 * half_ + 4; ++kk)
                                tc_mma_f16_ts(tb + 128, tb + kk * 8, mk(vb + kk * (2048 >> 4), HI), ATC_IDESC_PV, (j > 0 || kk > 0) ? 1u : 0u);
                            if (half_ && b == n_blocks - 1) tc_commit(&kv_empty[slot]);
                        }
                        __syncwarp();
                    }
                    if (!failed && j + 1 < n_tiles && !scores(b, j + 1)) failed = true;      // over P(j): the tensor core runs the product before it first
                }
            }
            if (!failed && leader) tc_commit(o_full);
        }
    } else if (warp < 4 * n_blocks) {
        // ===== softmax: thread = row
        const int blk = warp >> 2, r = tid - blk * AS_BLOCK, qi = (r0 + tid) / G;
        int lo = 0, hi = 0;
        if (tid < n_valid) {
            if (prefix) hi = e.cached;
            else {
                const int pos = e.cached + qi;
                hi = min(max(pos + 1, 0), table_end);
                lo = max(e.key_lo, a.window > pos ? 0 : pos - a.window + 1);
            }
        }
        const uint32_t ts = tmem + blk * 256 + ((uint32_t)((warp & 3) * 32) << 16), to_ = ts + 128;
        const float scale = a.scale_log2;
        float m_used = -INFINITY, m_true = -INFINITY, l = 0.f;
        int page = n_tiles > 0 ? page_of(0) : 0;
        for (int j = 0; j < n_tiles; ++j) {
            const int kb = key_tile(j) * AS_TK;
            const bool gone = page < 0;
            if (j + 1 < n_tiles) page = page_of(j + 1);
            if (!mbar_wait_warp(&s_full[blk], j & 1)) { failed = true; break; }
            tc_fence_after();
            // 32 scores at a time: the last two chunks are read twice, once for the maximum and again while the first ones are in work
            // (all 128 held through both passes take 230 registers)
            float x0[32], x1[32], x2[32];
            auto chunk_at = [&](int c, float (&x)[32]) { tc_ld32(ts + c * 32, x); };
            const bool clear = !gone && kb + AS_TK <= all_hi && (kb >= all_lo || kb + AS_TK <= sinks);
            auto mask = [&](int c, float (&x)[32]) {
                if (!clear) {
                    const int nh = (gone ? 0 : hi - kb) - c * 32, nl = lo - kb - c * 32, ns = sinks - kb - c * 32;
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = i < nh && (i >= nl || i < ns) ? x[i] : -INFINITY;
                }
            };
            float mx0 = -INFINITY, mx1 = -INFINITY;
            auto maximum = [&](const float (&x)[32]) {
                #pragma unroll
                for (int i = 0; i < 32; i += 4) { mx0 = fmax3(mx0, x[i], x[i + 1]); mx1 = fmax3(mx1, x[i + 2], x[i + 3]); }
            };
            chunk_at(2, x0); chunk_at(3, x1);
            tc_wait_ld();
            mask(2, x0); mask(3, x1);
            maximum(x0); maximum(x1);
            chunk_at(0, x0); chunk_at(1, x1);
            tc_wait_ld();
            mask(0, x0); mask(1, x1);
            maximum(x0); maximum(x1);
            m_true = fmaxf(m_true, fmaxf(mx0, mx1) * scale);                // raw scores: the scale is positive
            // the reference of the exponents moves only when the maximum has grown by 2^8, so O is seldom rescaled
            const bool move = m_true > m_used + ATC_RESCALE_THRESHOLD || (m_used == -INFINITY && m_true > -INFINITY);
            const bool rescale = move && m_used != -INFINITY;
            const float corr = rescale ? ex2_approx(m_used - m_true) : 1.0f;
            if (move) m_used = m_true;
            if (__any_sync(0xffffffffu, rescale)) {                         // O holds the tiles before: the scores came after their product
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float o[32];
                    tc_ld32(to_ + c * 32, o);
                    tc_wait_ld();
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= corr;
                    tc_st32(to_ + c * 32, o);
                }
            }
            // values that no row of the item sees may be anything (0 * NaN would spoil O): cleared by the first block, whose product comes
            // first, a key per thread
            if (blk == 0 && !gone && !(kb + AS_TK <= t.end && (kb >= t.lo || kb + AS_TK <= sinks))) {
                const int slot = (2 * j + 1) % SLOTS;
                if (!mbar_wait_sleep_warp(&kv_full[slot], ((2 * j + 1) / SLOTS) & 1)) { failed = true; break; }
                const int key = kb + r;
                if (!(key < t.end && (key >= t.lo || key < sinks))) {
                    #pragma unroll
                    for (int c = 0; c < 16; ++c)
                        *reinterpret_cast<uint4*>(smem + Cfg::OFF_KV + slot * AS_TILE + (c >> 3) * (AS_TILE / 2) + r * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
            }
            const float nref = m_used == -INFINITY ? 0.f : -m_used;
            const float2 scale2 = make_float2(scale, scale), nref2 = make_float2(nref, nref);
            float2 sum = make_float2(0.f, 0.f);
            uint32_t w[32];
            auto weights = [&](const float (&x)[32], int at) {
                #pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 y = fma2(make_float2(x[i], x[i + 1]), scale2, nref2);
                    const float2 ex = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                    sum = add2(sum, ex);
                    w[at + (i >> 1)] = pack_h2(ex.x, ex.y);                 // the one rounding of a weight, as the product takes it
                }
            };
            auto announce = [&](uint64_t* bar) {
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            chunk_at(2, x2);
            weights(x0, 0);
            weights(x1, 16);
            tc_st32u(ts, w);
            tc_wait_ld();
            announce(&p_half[blk]);
            chunk_at(3, x1);
            mask(2, x2);
            weights(x2, 0);
            tc_wait_ld();
            mask(3, x1);
            weights(x1, 16);
            tc_st32u(ts + 32, w);
            announce(&p_full[blk]);
            l = l * corr + (sum.x + sum.y);
        }
        // ===== O -> output or partial sum, by way of shared memory: a warp writes its 32 rows one after the other, each row whole
        failed = __any_sync(0xffffffffu, failed);
        if (!failed && n_tiles > 0 && !mbar_wait_sleep_warp(o_full, 0)) failed = true;
        if (!failed) {
            tc_fence_after();
            const bool direct = !prefix && e.key_lo == 0 && s_item.splits == 1;
            const float inv = direct ? (l > 0.f ? 1.0f / l : 0.f) : 1.0f;
            const int n_mine = min(32, n_valid - warp * 32);
            float* stage = reinterpret_cast<float*>(smem) + (size_t)tid * SPAN_PART;
            half* stage_h = reinterpret_cast<half*>(smem) + (size_t)tid * 136;          // rows of 272 bytes
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                float o[32];
                if (n_tiles > 0) { tc_ld32(to_ + c * 32, o); tc_wait_ld(); }
                else {
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.f;
                }
                if (direct) {
                    #pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<uint4*>(stage_h + c * 32 + i * 8) =
                            make_uint4(pack_h2(o[8 * i] * inv, o[8 * i + 1] * inv), pack_h2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                       pack_h2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack_h2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                } else {
                    #pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<float4*>(stage + c * 32 + 4 * i) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
            if (!direct) { stage[128] = m_used; stage[129] = l; }
            __syncwarp();
            if (direct) {
                for (int i = lane >> 4; i < n_mine; i += 2) {
                    const int pk = r0 + warp * 32 + i, q = pk / G;
                    reinterpret_cast<uint4*>(a.o)[((size_t)(e.row_base + q) * a.nq + kvh * G + (pk - q * G)) * 16 + (lane & 15)] =
                        *reinterpret_cast<const uint4*>(reinterpret_cast<const half*>(smem) + (size_t)(warp * 32 + i) * 136 + (lane & 15) * 8);
                }
            } else {
                for (int i = 0; i < n_mine; ++i) {
                    const int pk = r0 + warp * 32 + i, q = pk / G;
                    const float* from = reinterpret_cast<const float*>(smem) + (size_t)(warp * 32 + i) * SPAN_PART;
                    float* to = p.partial + (((size_t)s_item.split * a.rows + e.row_base + q) * a.nq + kvh * G + (pk - q * G)) * SPAN_PART;
                    reinterpret_cast<float4*>(to)[lane] = reinterpret_cast<const float4*>(from)[lane];
                    if (lane == 0) *reinterpret_cast<float2*>(to + 128) = *reinterpret_cast<const float2*>(from + 128);
                }
            }
        }
    }

    if (failed) s_failed = 1;
    tc_fence_before();
    __syncthreads();
    if (warp == SW + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::TMEM) : "memory");
    }
    if (tid == 0 && s_failed) atomicExch(p.status, 3);
    if (!p.first) pdl_wait();
}

// Joins the splits of the rows that attn_span_kernel computed alone: a warp per (row, head)
__global__ void __launch_bounds__(256) attn_span_join_kernel(const AsJoin p)
{
    pdl_enter();
    const SpanArgs& a = p.a;
    const int lane = threadIdx.x & 31, G = a.nq / a.nkv;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= (long long)a.rows * a.nq) return;
    const int row = (int)(w / a.nq);
    int b;
    if (a.cu_q) {
        int lo = 0, hi = a.bsz;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.cu_q[mid] <= row) lo = mid; else hi = mid; }
        b = lo;
    } else b = row / a.q_len;
    const SpanSeq s = span_seq(a, b);
    if (row < s.row_base || row >= s.row_base + s.ql || s.ql * G <= AR_ROWS) return;
    const SpanGroup g = span_group(a, b, s.cached);
    const int own = as_splits(as_own_tiles(a, s, g.len, G, p.own_rows), *p.own_chunk);
    if (own == 1 && g.g < 0) return;                         // written already
    const int pre = g.g < 0 ? 0 : as_splits((g.len + AS_TK - 1) / AS_TK, *p.prefix_chunk);
    AsSum sum = {make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f};
    const size_t step = (size_t)a.rows * a.nq * SPAN_PART;
    #pragma unroll 4
    for (int i = 0; i < pre; ++i) as_add(sum, p.prefix + w * SPAN_PART + i * step, lane);
    #pragma unroll 4
    for (int i = 0; i < own; ++i) as_add(sum, p.own + w * SPAN_PART + i * step, lane);
    const float inv = sum.l > 0.f ? 1.0f / sum.l : 0.f;
    reinterpret_cast<uint2*>(a.o)[w * 32 + lane] = make_uint2(pack_h2(sum.acc.x * inv, sum.acc.y * inv), pack_h2(sum.acc.z * inv, sum.acc.w * inv));
}

}  // namespace exl3
