// Attention over spans of the cache on tcgen05: sequences with more than 16 (query, head) rows per kv head, and the shared prefixes, whose
// rows are those of all sequences of a group.
//
// An item is 128 packed rows of one kv head and a run of key tiles of 128.  S = Q K^T (128 x 128) and O += P V are 128-column accumulators
// in tensor memory, P goes back over the first half of S as packed fp16 and is the A operand of the second product.  One softmax thread
// owns a row, so maxima and sums need no exchange.
//
// What bounds it: per tile and row block 776 + 512 cycles of the tensor core (128 x 128 x 16 with A in shared memory takes 97 cycles, in
// tensor memory 64), 1024 of the special-function unit (16 exponentials per clock and SM), in a chain of scores, softmax, product that one
// CTA cannot overlap with itself.  So two CTAs share an SM - 97 KB of shared memory, 256 columns and 192 threads each - and one's
// softmax runs under the other's products; the start and end of items overlap in the same way.
//
// Items are found by every CTA from the lengths themselves (warp 0, entries over lanes), which costs about a microsecond under the other
// CTA's work and saves a launch in front.  A run of tiles is cut into as many splits as fill the GPU, by the same rule in every CTA.
#pragma once
#include "attn_rows.cuh"
#include "attn_tc_ops.cuh"

namespace exl3 {

constexpr int AS_ROWS = 128;
constexpr int AS_THREADS = 192;                         // 4 softmax warps, TMA producer, MMA issuer
constexpr int AS_TILE = AS_TK * 256;                    // bytes of a tile of K, V or Q: two 64-dim halves of 16 KB
constexpr int AS_OFF_Q = 0, AS_OFF_K = AS_TILE, AS_OFF_V = 2 * AS_TILE, AS_OFF_BAR = 3 * AS_TILE;
constexpr int AS_NBARS = 8;                             // q_full, k_full, k_empty, v_full, v_empty, s_full, p_full, o_full
constexpr int AS_SMEM = AS_OFF_BAR + AS_NBARS * 8 + 16 + 1024;
constexpr int AS_MAX_SPLITS = 32;
constexpr int AS_ITEM_COST = 4;                         // start and end of an item, in tiles
static_assert(AS_ROWS * AR_MS * 4 <= 3 * AS_TILE, "partial sums are staged over the tiles");
static_assert(2 * (AS_SMEM + 1024) <= EXL3_SM_SMEM, "two CTAs per SM");

struct AsParams {
    SpanArgs a;
    float* partial;                                     // [2 * max_splits][rows][nq][AR_MS]: splits of the prefix, then a sequence's own
    int* chunk;                                         // key tiles per split, for the kernels behind
    int* status;
    int max_splits, own_base;                           // where a sequence's own splits begin among the partial sums
    int max_items, slots, n_seqs;           // n_seqs: 0 where no sequence has more than 16 rows
};

// A run of rows over one run of keys, before it is cut into items: prefix entries first, then sequences
struct AsEntry { int tab, row_base, n_rows, ql, cached, key_lo, prefix, tiles; };

__device__ __forceinline__ int as_blocks(int packed) { return (packed + AS_ROWS - 1) / AS_ROWS; }
// tiles of a sequence's last row block, which has as many as any other but for alignment
__device__ __forceinline__ int as_own_tiles(const SpanArgs& a, const SpanSeq& s, int key_lo, int G)
{
    const int i_first = (as_blocks(s.ql * G) - 1) * AS_ROWS / G;
    const SpanTiles t = span_tiles<AS_TK>(a, s.cached + i_first, s.cached + s.ql - 1, key_lo);
    return t.sink + t.near;
}
__device__ __forceinline__ AsEntry as_entry(const SpanArgs& a, int e, int G)
{
    AsEntry r = {0, 0, 0, 0, 0, 0, 0, 0};
    if (e < a.n_groups) {
        const int first = max(a.group_start[e], 0), last = min(a.group_start[e + 1], a.bsz);
        const int len = min(a.prefix_lens[e], a.pps * EXL3_PAGE);
        if (first >= last || len <= 0) return r;
        const int r0 = max(a.cu_q ? a.cu_q[first] : first * a.q_len, 0), r1 = min(a.cu_q ? a.cu_q[last] : last * a.q_len, a.rows);
        if (r0 >= r1) return r;
        r.tab = first; r.row_base = r0; r.ql = r1 - r0; r.prefix = len; r.tiles = (len + AS_TK - 1) / AS_TK;
    } else {
        const int b = e - a.n_groups;
        const SpanSeq s = span_seq(a, b);
        if (s.ql * G <= AR_ROWS) return r;
        r.tab = b; r.row_base = s.row_base; r.ql = s.ql; r.cached = s.cached;
        r.key_lo = span_group(a, b, s.cached).len;
        r.tiles = as_own_tiles(a, s, r.key_lo, G);
    }
    r.n_rows = r.ql * G;
    return r;
}

struct AsItem { AsEntry e; int rb, split, splits, kvh; };

// The item of this CTA (warp-uniform, all lanes); false: there is none.  chunk: tiles per split, as all CTAs find it.
__device__ __forceinline__ bool as_item(const AsParams& p, int G, int lane, AsItem& it, int& chunk)
{
    const SpanArgs& a = p.a;
    const int n = a.n_groups + p.n_seqs;
    int most = 1;
    for (int e0 = 0; e0 < n; e0 += 32)
        if (e0 + lane < n) most = max(most, as_entry(a, e0 + lane, G).tiles);
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    // lane i weighs i + 1 splits of the longest run: waves of items times what an item takes
    const int mine = (most + lane) / (lane + 1);
    long long items = 0;
    for (int e0 = 0; e0 < n; e0 += 32) {
        AsEntry e = {};
        if (e0 + lane < n) e = as_entry(a, e0 + lane, G);
        const int units = as_blocks(e.n_rows) * a.nkv;
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
    int before = 0;
    for (int e0 = 0; e0 < n; e0 += 32) {
        AsEntry e = {};
        if (e0 + lane < n) e = as_entry(a, e0 + lane, G);
        const int rb = as_blocks(e.n_rows), sp = as_splits(e.tiles, chunk), own = rb * a.nkv * sp;
        int v = own;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += u; }
        const int at = (int)blockIdx.x - before;
        const unsigned behind = __ballot_sync(0xffffffffu, v > at);
        if (behind) {
            const int j = __ffs(behind) - 1;
            const int in = at - __shfl_sync(0xffffffffu, v - own, j), n_rb = __shfl_sync(0xffffffffu, rb, j);
            it.splits = __shfl_sync(0xffffffffu, sp, j);
            it.e = as_entry(a, e0 + j, G);
            // row blocks of a head and run are neighbours, which read the same keys; the last, the longest where it is causal, first
            it.rb = n_rb - 1 - in % n_rb; it.split = in / n_rb % it.splits; it.kvh = in / n_rb / it.splits;
            return true;
        }
        before += __shfl_sync(0xffffffffu, v, 31);
    }
    return false;
}

__global__ void __launch_bounds__(AS_THREADS, 2) attn_span_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                  const AsParams p, int early)
{
    (void)early;
    pdl_wait();
    extern __shared__ uint8_t smem_unaligned[];
    uint8_t* smem = smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + AS_OFF_BAR);
    uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 2, *v_full = bars + 3, *v_empty = bars + 4, *s_full = bars + 5, *p_full = bars + 6,
             *o_full = bars + 7;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + AS_NBARS);
    __shared__ AsItem s_item;
    __shared__ int s_have, s_failed;

    const SpanArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.nq / a.nkv;
    if (warp == 0) {
        AsItem it;
        int chunk;
        const bool have = as_item(p, G, lane, it, chunk);
        if (lane == 0) {
            s_have = have; s_item = it; s_failed = 0;
            if (blockIdx.x == 0) *p.chunk = chunk;
        }
    }
    if (tid == 32) {
        mbar_init(q_full, 4); mbar_init(p_full, 4);
        mbar_init(k_full, 1); mbar_init(k_empty, 1); mbar_init(v_full, 1); mbar_init(v_empty, 1); mbar_init(s_full, 1); mbar_init(o_full, 1);
        mbar_fence_init();
    }
    __syncthreads();
    if (!s_have) return;
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(256) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    const AsEntry e = s_item.e;
    const int kvh = s_item.kvh, r0 = s_item.rb * AS_ROWS, n_valid = min(AS_ROWS, e.n_rows - r0);
    const int table_end = a.pps * EXL3_PAGE;
    const int i_first = r0 / G, i_last = (r0 + n_valid - 1) / G;
    // the block's key tiles, and this item's part [t0, t1) of them
    SpanTiles t;
    int all_lo, all_hi, sinks;                              // what every row of the block sees
    if (e.prefix) {
        t.sink = 0; t.first = 0; t.near = e.tiles; t.lo = 0; t.end = e.prefix;
        all_lo = 0; all_hi = e.prefix; sinks = 0;
    } else {
        const int p_first = e.cached + i_first, p_last = e.cached + i_last;
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

    if (warp < 4) {
        // the Q row of every softmax thread -> shared memory, K-major, 128-byte swizzle
        const int pr = r0 + tid, qi = pr / G;
        const uint4* src = reinterpret_cast<const uint4*>(a.q + ((size_t)(e.row_base + qi) * a.nq + kvh * G + (pr - qi * G)) * 128);
        #pragma unroll
        for (int c = 0; c < 16; ++c) {
            const uint4 x = tid < n_valid ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(smem + AS_OFF_Q + (c >> 3) * (AS_TILE / 2) + tid * 128 + (((c & 7) ^ (tid & 7)) << 4)) = x;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // kernels behind may be set up from here on (in front of the allocation they could take the tensor memory and wait for this one)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = *tmem_slot, tmem_o = tmem + 128;
    bool failed = false;

    if (warp == 4) {
        // ===== producer
        if (lane == 0 && n_tiles > 0) {
            int page = page_of(0), asked_k = 0, asked_v = 0;
            for (int j = 0; j < n_tiles; ++j) {
                const int tok = (key_tile(j) * AS_TK) & (EXL3_PAGE - 1);
                const int pg = page < 0 ? a.pages : page;   // outside the pool: zeros, which the softmax threads mask
                if (j + 1 < n_tiles) page = page_of(j + 1);
                if (j > 0 && !mbar_wait_sleep(k_empty, (j - 1) & 1)) { failed = true; break; }
                mbar_expect_tx(k_full, AS_TILE);
                tma_load_5d(smem + AS_OFF_K, &kmap, 0, tok, 0, kvh, pg, k_full);
                ++asked_k;
                if (j > 0 && !mbar_wait_sleep(v_empty, (j - 1) & 1)) { failed = true; break; }
                mbar_expect_tx(v_full, AS_TILE);
                tma_load_5d(smem + AS_OFF_V, &vmap, 0, tok, 0, kvh, pg, v_full);
                ++asked_v;
            }
            // not out before every copy has landed, whatever became of those who take them
            if (asked_k > 0) mbar_wait_sleep(k_full, (asked_k - 1) & 1);
            if (asked_v > 0) mbar_wait_sleep(v_full, (asked_v - 1) & 1);
        }
    } else if (warp == 5) {
        // ===== MMA issuer: warp-uniform values, one elected lane
        if (n_tiles > 0) {
            const bool leader = elect_one();
            constexpr uint32_t HI = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);     // SBO, version 1, SWIZZLE_128B
            constexpr uint32_t LBO_K = 1u << 16, LBO_V = (uint32_t)((AS_TILE / 2) >> 4) << 16;
            auto mk = [](uint32_t lo, uint32_t hi) { return ((uint64_t)hi << 32) | lo; };
            const uint32_t q_lo = (smem_u32(smem + AS_OFF_Q) >> 4) | LBO_K, k_lo = (smem_u32(smem + AS_OFF_K) >> 4) | LBO_K;
            const uint32_t v_lo = (smem_u32(smem + AS_OFF_V) >> 4) | LBO_V;
            auto scores = [&](int j) -> bool {
                if (!mbar_wait_sleep_warp(k_full, j & 1)) return false;
                tc_fence_after();
                if (leader) {
                    #pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t off = ((kk >> 2) * (AS_TILE / 2) + (kk & 3) * 32) >> 4;
                        tc_mma_f16(tmem, mk(q_lo + off, HI), mk(k_lo + off, HI), ATC_IDESC_S, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(s_full);
                    tc_commit(k_empty);
                }
                __syncwarp();
                return true;
            };
            if (!mbar_wait_sleep_warp(q_full, 0) || !scores(0)) failed = true;
            for (int j = 0; j < n_tiles && !failed; ++j) {
                if (!mbar_wait_warp(p_full, j & 1) || !mbar_wait_sleep_warp(v_full, j & 1)) { failed = true; break; }
                tc_fence_after();
                if (leader) {
                    #pragma unroll
                    for (int kk = 0; kk < 8; ++kk)
                        tc_mma_f16_ts(tmem_o, tmem + kk * 8, mk(v_lo + kk * (2048 >> 4), HI), ATC_IDESC_PV, (j > 0 || kk > 0) ? 1u : 0u);
                    tc_commit(v_empty);
                }
                __syncwarp();
                if (j + 1 < n_tiles && !scores(j + 1)) failed = true;      // over P(j): the tensor core runs the product before it first
            }
            if (!failed && leader) tc_commit(o_full);
        }
    } else {
        // ===== softmax: thread = row
        const int qi = (r0 + tid) / G;
        const bool valid = tid < n_valid;
        int lo = 0, hi = 0;
        if (valid) {
            if (e.prefix) hi = e.prefix;
            else {
                const int pos = e.cached + qi;
                hi = min(max(pos + 1, 0), table_end);
                lo = max(e.key_lo, a.window > pos ? 0 : pos - a.window + 1);
            }
        }
        const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
        const float scale = a.scale_log2;
        float m_used = -INFINITY, m_true = -INFINITY, l = 0.f;
        int page = n_tiles > 0 ? page_of(0) : 0;
        for (int j = 0; j < n_tiles; ++j) {
            const int kb = key_tile(j) * AS_TK;
            const bool gone = page < 0;
            if (j + 1 < n_tiles) page = page_of(j + 1);
            if (!mbar_wait_warp(s_full, j & 1)) { failed = true; break; }
            tc_fence_after();
            float s[AS_TK];
            #pragma unroll
            for (int c = 0; c < 4; ++c) tc_ld32(tmem + lane_addr + c * 32, *reinterpret_cast<float (*)[32]>(&s[c * 32]));
            tc_wait_ld();
            const bool clear = !gone && kb + AS_TK <= all_hi && (kb >= all_lo || kb + AS_TK <= sinks);
            if (!clear) {
                const int nh = gone ? 0 : hi - kb, nl = lo - kb, ns = sinks - kb;
                #pragma unroll
                for (int i = 0; i < AS_TK; ++i) s[i] = i < nh && (i >= nl || i < ns) ? s[i] : -INFINITY;
            }
            float mx0 = -INFINITY, mx1 = -INFINITY;
            #pragma unroll
            for (int i = 0; i < AS_TK; i += 4) { mx0 = fmax3(mx0, s[i], s[i + 1]); mx1 = fmax3(mx1, s[i + 2], s[i + 3]); }
            m_true = fmaxf(m_true, fmaxf(mx0, mx1) * scale);                // raw scores: the scale is positive
            // the reference of the exponents moves only when the maximum has grown by 2^8, so O is seldom rescaled
            const bool move = m_true > m_used + ATC_RESCALE_THRESHOLD || (m_used == -INFINITY && m_true > -INFINITY);
            const bool rescale = move && m_used != -INFINITY;
            const float corr = rescale ? ex2_approx(m_used - m_true) : 1.0f;
            if (move) m_used = m_true;
            const float nref = m_used == -INFINITY ? 0.f : -m_used;
            float l0 = 0.f, l1 = 0.f;
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t w[32];
                #pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const float e0 = ex2_approx(fmaf(s[c * 64 + i], scale, nref)), e1 = ex2_approx(fmaf(s[c * 64 + i + 1], scale, nref));
                    l0 += e0; l1 += e1;
                    w[i >> 1] = pack_h2(e0, e1);                            // the one rounding of a weight, as the product takes it
                }
                tc_st32u(tmem + lane_addr + c * 32, w);
            }
            l = l * corr + (l0 + l1);
            if (__any_sync(0xffffffffu, rescale)) {                         // O holds the tiles before: the scores came after their product
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float o[32];
                    tc_ld32(tmem_o + lane_addr + c * 32, o);
                    tc_wait_ld();
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= corr;
                    tc_st32(tmem_o + lane_addr + c * 32, o);
                }
            }
            // values that no row of the block sees may be anything (0 * NaN would spoil O): cleared, a key per thread
            if (!gone && !(kb + AS_TK <= t.end && (kb >= t.lo || kb + AS_TK <= sinks))) {
                if (!mbar_wait_sleep_warp(v_full, j & 1)) { failed = true; break; }
                const int key = kb + tid;
                if (!(key < t.end && (key >= t.lo || key < sinks))) {
                    #pragma unroll
                    for (int c = 0; c < 16; ++c)
                        *reinterpret_cast<uint4*>(smem + AS_OFF_V + (c >> 3) * (AS_TILE / 2) + tid * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
        }
        // ===== O -> output or partial sum, by way of shared memory: a warp writes its 32 rows one after the other, each row whole
        failed = __any_sync(0xffffffffu, failed);
        if (!failed && n_tiles > 0 && !mbar_wait_sleep_warp(o_full, 0)) failed = true;
        if (!failed) {
            tc_fence_after();
            const bool direct = !e.prefix && e.key_lo == 0 && s_item.splits == 1;
            const float inv = direct ? (l > 0.f ? 1.0f / l : 0.f) : 1.0f;
            const int n_mine = min(32, n_valid - warp * 32);
            float* stage = reinterpret_cast<float*>(smem) + (size_t)tid * AR_MS;
            half* stage_h = reinterpret_cast<half*>(smem) + (size_t)tid * 136;          // rows of 272 bytes
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                float o[32];
                if (n_tiles > 0) { tc_ld32(tmem_o + lane_addr + c * 32, o); tc_wait_ld(); }
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
                for (int r = lane >> 4; r < n_mine; r += 2) {
                    const int pk = r0 + warp * 32 + r, i = pk / G;
                    reinterpret_cast<uint4*>(a.o)[((size_t)(e.row_base + i) * a.nq + kvh * G + (pk - i * G)) * 16 + (lane & 15)] =
                        *reinterpret_cast<const uint4*>(reinterpret_cast<const half*>(smem) + (size_t)(warp * 32 + r) * 136 + (lane & 15) * 8);
                }
            } else {
                const size_t split = (size_t)(e.prefix ? 0 : p.own_base) + s_item.split;
                for (int r = 0; r < n_mine; ++r) {
                    const int pk = r0 + warp * 32 + r, i = pk / G;
                    const float* from = reinterpret_cast<const float*>(smem) + (size_t)(warp * 32 + r) * AR_MS;
                    float* to = p.partial + ((split * a.rows + e.row_base + i) * a.nq + kvh * G + (pk - i * G)) * AR_MS;
                    reinterpret_cast<float4*>(to)[lane] = reinterpret_cast<const float4*>(from)[lane];
                    if (lane == 0) *reinterpret_cast<float2*>(to + 128) = *reinterpret_cast<const float2*>(from + 128);
                }
            }
        }
    }

    if (failed) s_failed = 1;
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
    }
    if (tid == 0 && s_failed) atomicExch(p.status, 3);
}

// Joins the splits of the rows that attn_span_kernel computed alone: a warp per (row, head)
__global__ void __launch_bounds__(256) attn_span_join_kernel(const AsParams p)
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
    const int chunk = *p.chunk, own = as_splits(as_own_tiles(a, s, g.len, G), chunk);
    if (own == 1 && g.g < 0) return;                         // written already
    const int pre = g.g < 0 ? 0 : as_splits((g.len + AS_TK - 1) / AS_TK, chunk);
    AsSum sum = {make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f};
    const size_t step = (size_t)a.rows * a.nq * AR_MS;
    const float* base = p.partial + w * AR_MS;
    #pragma unroll 4
    for (int i = 0; i < pre; ++i) as_add(sum, base + i * step, lane);
    #pragma unroll 4
    for (int i = 0; i < own; ++i) as_add(sum, base + (p.own_base + i) * step, lane);
    const float inv = sum.l > 0.f ? 1.0f / sum.l : 0.f;
    reinterpret_cast<uint2*>(a.o)[w * 32 + lane] = make_uint2(pack_h2(sum.acc.x * inv, sum.acc.y * inv), pack_h2(sum.acc.z * inv, sum.acc.w * inv));
}

}  // namespace exl3
