// Attention over spans of the cache on tcgen05: sequences with more than 16 (query, head) rows per kv head, and the shared prefixes, whose
// rows are those of all sequences of a group.
//
// A unit is NB blocks of 128 packed rows of one kv head and the key tiles of 128 that they see.  S = Q K^T (128 x 128) and O += P V are
// 128-column accumulators in tensor memory per block, P goes back over the first half of S as packed fp16 and is the A operand of the
// second product.  One softmax thread owns a row, so maxima and sums need no exchange.
//
// What bounds it: per tile and row block 776 + 512 cycles of the tensor core (128 x 128 x 16 with A in shared memory takes 97 cycles, in
// tensor memory 64), 1024 of the special-function unit (16 exponentials per clock and SM) and 64 KB of keys and values out of L2, in a
// chain of scores, softmax, product that a block cannot overlap with itself.  So an SM holds two blocks, whose softmax runs under the
// other's products: NB = 2, one CTA whose blocks share every tile, where sequences have the rows (with two CTAs that read tiles of their own
// 4 x 2048 rows took 794 us: 64 KB per 2500 cycles and SM is what L2 gives); NB = 1, two CTAs of one block, where they do not, so that
// the start and end of short units overlap.  4 x 2048 rows over windows of 4096, 40 / 8 heads: 736 to 750 us, 800 to 820 TFLOP/s; 8 x 128 rows over
// 32768 shared keys and up to 300 of their own, 690 GFLOP, with the join: 872 to 882 us, 780 to 790 TFLOP/s.  (Tried on an earlier build: a
// quarter or a sixth of the exponentials by a polynomial 728 and 720 us for 725, so they are not what a tile waits for; P announced after 96
// keys instead of 64 710 for 712 and, over shared keys, 893 for 846.)
//
// Queries come as copies of whole rows, a unit ahead: a unit has rows * G <= 128 NB packed rows (read by the softmax threads at a unit's
// start instead: 4 x 2048 rows 779 us).
//
// The tiles of all units stand in one line, of which every CTA takes an equal part (one item per CTA, with the splits chosen for the fewest
// waves, left SMs idle for 30 % of 8 x 128 rows over a shared prefix: 160 units on 148 SMs).  The parts are found from the lengths by each
// CTA itself, which costs about two microseconds once and saves a launch in front.  A unit cut by the border of a part goes through
// partial sums: of a prefix they stay for span_join_kernel, which adds them to each sequence's own; of a sequence's own span the warp that
// arrives last with its 32 rows adds them up in the order of the parts.
#pragma once
#include "attn_rows.cuh"
#include "attn_tc_ops.cuh"

namespace exl3 {

constexpr int AS_BLOCK = 128;                            // rows of a block: the lanes of tensor memory
constexpr int AS_TILE = AS_TK * 256;                    // bytes of a tile of K, V or Q: two 64-dim halves of 16 KB
constexpr int AS_MAX_SPLITS = 32;
constexpr int AS_MAX_CHUNKS = 256;                      // of 32 sequences
// An exponent is one fused score * scale - reference, whose product is not rounded, against a reference that is: off by half a step of the
// reference, for all keys of a part of a row alike but not for its other parts, and from 2^28 on by more than fp16 weights hold (they came out
// infinite, the output NaN).  Where a reference is this far from 0, where half a step is 2^-12, the maximum is subtracted ahead of the scale.
constexpr float AS_FAR = 8192.0f;

// A unit's part in work, as the producer finds it
struct AsPiece {
    int n_tiles;                                        // 0: there are no more
    int t0, sink, first, lo, end, any;                  // tiles t0.. of the unit's, which are `sink` from key tile 0 on, then those from `first` on; any: there are some
    int all_lo, all_hi, sinks;                          // keys that every row sees
    int tab, row_base, r0, n_valid, cached, key_lo, kvh;
    int ring;                                           // number of its first K tile in the ring
    int index, count, c0;                               // number among the unit's parts, their count, the CTA of the first
    int group;                                          // >= 0: a prefix is added
};

template <int NB>
struct AsCfg {
    static constexpr int ROWS = AS_BLOCK * NB, SW = 4 * NB, THREADS = (SW + 2) * 32;       // softmax warps, TMA producer, MMA issuer
    static constexpr int SLOTS = 2 * NB;                                                   // ring of tiles: K0 V0 K1 V1 ...
    static constexpr int QHALF = ROWS * 128;                                               // Q: halves of a head, rows of 128 bytes
    static constexpr int OFF_KV = NB * AS_TILE, OFF_STAGE = OFF_KV + SLOTS * AS_TILE;      // Q in front; 2 KB per softmax warp
    static constexpr int OFF_PIECE = OFF_STAGE + SW * 2048;
    static constexpr int OFF_SUM = OFF_PIECE + 2 * (int)sizeof(AsPiece);
    static constexpr int OFF_BAR = OFF_SUM + (AS_MAX_CHUNKS + 2) * 4;
    static constexpr int NBARS = 4 * NB + 2 * SLOTS + 6;                                   // s_full, p_half, p_full, o_full; full, empty per slot; piece full, empty; q full, empty
    static constexpr int SMEM = OFF_BAR + NBARS * 8 + 16 + 1024;
    static constexpr int CTAS = NB == 1 ? 2 : 1, TMEM = 256 * NB;
    static_assert(OFF_SUM % 8 == 0 && OFF_BAR % 8 == 0, "alignment of the barriers");
    static_assert(CTAS * (SMEM + 1024 + 64) <= EXL3_SM_SMEM, "CTAs of an SM");
};

struct AsParams {
    SpanArgs a;
    int prefixes;                                       // 1: the groups' prefixes, 0: the sequences' own spans
    float* partial;                                     // prefixes: [splits][rows][nq][SPAN_PART]; own spans: [2 * CTAs][SW][32 * SPAN_PART]
    int* share;                                         // tiles per CTA, for the kernels behind (0: units are not cut)
    int max_splits;
    float* rest;                                        // own spans: [rows][nq][SPAN_PART] partial sums of sequences that a prefix is added to
    int* counters;                                      // own spans: [CTAs][SW], zero between calls
    int* status;
    int first;                                          // nothing of this call is in front of the launch
};

// A run of rows over one run of keys: a group over its prefix, a sequence over its own span
struct AsEntry { int tab, row_base, n_rows, cached, key_lo, group; };

__device__ __forceinline__ int as_blocks(int packed, int rows) { return (packed + rows - 1) / rows; }
__device__ __forceinline__ AsEntry as_entry(const AsParams& p, int e, int G)
{
    const SpanArgs& a = p.a;
    AsEntry r = {0, 0, 0, 0, 0, -1};
    if (p.prefixes) {
        const int first = max(a.group_start[e], 0), last = min(a.group_start[e + 1], a.bsz);
        const int len = min(a.prefix_lens[e], a.pps * EXL3_PAGE);
        if (first >= last || len <= 0) return r;
        const int r0 = max(a.cu_q ? a.cu_q[first] : first * a.q_len, 0), r1 = min(a.cu_q ? a.cu_q[last] : last * a.q_len, a.rows);
        if (r0 >= r1) return r;
        r.tab = first; r.row_base = r0; r.cached = len; r.n_rows = (r1 - r0) * G;
    } else {
        const SpanSeq s = span_seq(a, e);
        if (s.ql * G <= AR_ROWS) return r;
        const SpanGroup g = span_group(a, e, s.cached);
        r.tab = e; r.row_base = s.row_base; r.cached = s.cached; r.key_lo = g.len; r.group = g.g; r.n_rows = s.ql * G;
    }
    return r;
}
// the key tiles of an entry's rows [r0, r1)
__device__ __forceinline__ SpanTiles as_tiles(const AsParams& p, const AsEntry& e, int r0, int r1, int G)
{
    if (p.prefixes) { SpanTiles t = {0, 0, (e.cached + AS_TK - 1) / AS_TK, 0, e.cached}; return t; }
    return span_tiles<AS_TK>(p.a, e.cached + r0 / G, e.cached + (r1 - 1) / G, e.key_lo);
}
__device__ __forceinline__ int as_count(const AsParams& p, const AsEntry& e, int rb, int rows, int G)
{
    const SpanTiles t = as_tiles(p, e, rb * rows, min(rb * rows + rows, e.n_rows), G);
    return max(t.sink + t.near, 1);                     // a unit whose rows see nothing is there all the same: its output is written
}
// tiles of the row blocks [rb0, rb1) of an entry that all lanes have
__device__ __forceinline__ int as_sum_blocks(const AsParams& p, const AsEntry& e, int rb0, int rb1, int rows, int G, int lane)
{
    int v = 0;
    for (int rb = rb0 + lane; rb < rb1; rb += 32) v += as_count(p, e, rb, rows, G);
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ AsEntry as_shfl(const AsEntry& e, int j)
{
    AsEntry r;
    r.tab = __shfl_sync(0xffffffffu, e.tab, j); r.row_base = __shfl_sync(0xffffffffu, e.row_base, j); r.n_rows = __shfl_sync(0xffffffffu, e.n_rows, j);
    r.cached = __shfl_sync(0xffffffffu, e.cached, j); r.key_lo = __shfl_sync(0xffffffffu, e.key_lo, j); r.group = __shfl_sync(0xffffffffu, e.group, j);
    return r;
}
// tiles per head of entry e0 + lane, which is returned too
__device__ __forceinline__ int as_entry_tiles(const AsParams& p, int e0, int n, int rows, int G, int lane, AsEntry& e)
{
    e = {0, 0, 0, 0, 0, -1};
    if (e0 + lane < n) e = as_entry(p, e0 + lane, G);
    const int n_rb = as_blocks(e.n_rows, rows);
    if (p.prefixes) return n_rb * ((e.cached + AS_TK - 1) / AS_TK);
    int v = 0;
    if (n_rb <= 4)
        for (int rb = 0; rb < n_rb; ++rb) v += as_count(p, e, rb, rows, G);
    unsigned wide = __ballot_sync(0xffffffffu, n_rb > 4);
    while (wide) {
        const int j = __ffs(wide) - 1;
        wide &= wide - 1;
        const AsEntry x = as_shfl(e, j);
        const int sum = as_sum_blocks(p, x, 0, as_blocks(x.n_rows, rows), rows, G, lane);
        if (lane == j) v = sum;
    }
    return v;
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

// BESIDE: the kernel of few rows runs at the same time (a kernel of its own: the code for it cost calls without it 1 to 2 us)
template <int NB, bool BESIDE>
__global__ void __launch_bounds__(AsCfg<NB>::THREADS, AsCfg<NB>::CTAS) attn_span_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                                         const __grid_constant__ CUtensorMap vmap,
                                                                                         const __grid_constant__ CUtensorMap qmap,
                                                                                         const AsParams p, int early)
{
    using Cfg = AsCfg<NB>;
    constexpr int SW = Cfg::SW, SLOTS = Cfg::SLOTS;
    (void)early;
    pdl_wait();
    extern __shared__ uint8_t smem_unaligned[];
    uint8_t* smem = smem_unaligned + ((1024u - (smem_u32(smem_unaligned) & 1023u)) & 1023u);
    AsPiece* pieces = reinterpret_cast<AsPiece*>(smem + Cfg::OFF_PIECE);
    int* sums = reinterpret_cast<int*>(smem + Cfg::OFF_SUM);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
    uint64_t *s_full = bars, *p_half = s_full + NB, *p_full = p_half + NB, *o_full = p_full + NB, *kv_full = o_full + NB,
             *kv_empty = kv_full + SLOTS, *piece_full = kv_empty + SLOTS, *piece_empty = piece_full + 2, *q_full = piece_empty + 2, *q_empty = q_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::NBARS);
    __shared__ int s_failed;
    __shared__ SpanLoad loads[BESIDE ? SW + 2 : 1];

    const SpanArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.nq / a.nkv, n = p.prefixes ? a.n_groups : a.bsz, n_chunks = (n + 31) / 32;
    const int rows = Cfg::ROWS / G * G;                     // of a unit: whole rows of the call, so that a copy places them as packed rows
    if (tid == 0) {
        s_failed = 0;
        mbar_init(q_full, 1); mbar_init(q_empty, 1);
        for (int i = 0; i < NB; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_half[i], 4); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1); }
        for (int i = 0; i < SLOTS; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&piece_full[i], 1); mbar_init(&piece_empty[i], SW + 1); }
        mbar_fence_init();
    }
    // the line's length: tiles of every 32 sequences, longest unit
    int longest = 0;
    SpanLoad load = {0, 0};
    AsEntry mine = {0, 0, 0, 0, 0, -1};                     // of the first chunk, which the producer keeps
    int tiles = 0;
    for (int ch = (warp + 2) % (SW + 2); ch < n_chunks; ch += SW + 2) {
        AsEntry e;
        const int own = as_entry_tiles(p, ch * 32, n, rows, G, lane, e);
        if (ch == 0) { mine = e; tiles = own; }
        int v = own;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) sums[ch] = v;
        if (p.prefixes) longest = max(longest, (e.cached + AS_TK - 1) / AS_TK);
        else if (BESIDE && ch * 32 + lane < n) span_load(a, ch * 32 + lane, AR_ROWS, load);
    }
    if (BESIDE) span_load_put(loads, warp, load, lane);
    if (p.prefixes) {
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
        if (lane == 0 && tid == 0) sums[AS_MAX_CHUNKS] = 0;
        __syncthreads();
        if (lane == 0) atomicMax(&sums[AS_MAX_CHUNKS], longest);
    }
    __syncthreads();
    long long F = 0;
    for (int ch = lane; ch < n_chunks; ch += 32) F += sums[ch];
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) F += __shfl_xor_sync(0xffffffffu, F, o);
    F *= a.nkv;
    const int ctas = BESIDE ? max(Cfg::CTAS * (a.beside - span_few_sms(a, loads, SW + 2)), 1) : gridDim.x;
    long long share = max((F + ctas - 1) / ctas, 1LL);
    // a prefix's parts each have a place among the partial sums; with one place units stay whole, with the CTA where they begin
    const bool cut = !p.prefixes || p.max_splits > 1;
    if (p.prefixes && p.max_splits > 2) share = max(share, (long long)(sums[AS_MAX_CHUNKS] - 1) / (p.max_splits - 1) + 1);
    else if (p.prefixes && cut) share = max(share, (long long)sums[AS_MAX_CHUNKS]);
    const long long f0 = min(blockIdx.x * share, F), f1 = min(f0 + share, F);
    if (blockIdx.x == 0 && tid == 0) *p.share = cut ? (int)min(share, 1LL << 30) : 0;
    if (f0 >= f1) return;
    if (warp == SW + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Cfg::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // kernels behind may be set up from here on (in front of the allocation they could take the tensor memory and wait for this one)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    bool failed = false;

    if (warp == SW) {
        // ===== producer: walks this CTA's part of the line; warp-uniform, lane 0 issues
        int ch = 0, it = 0, n_piece = 0, n_q = 0;
        long long f = f0, at = 0;                           // at: where the chunk, then the entry begins
        while ((long long)(sums[ch] * (long long)a.nkv) + at <= f) { at += sums[ch] * (long long)a.nkv; ++ch; }
        if (ch > 0) tiles = as_entry_tiles(p, ch * 32, n, rows, G, lane, mine);
        int j = 0;                                          // entry of the chunk
        auto seek = [&]() {                                  // entry j of the chunk that has f
            while (true) {
                const long long w = (long long)__shfl_sync(0xffffffffu, tiles, j) * a.nkv;
                if (at + w > f) return;
                at += w;
                if (++j == 32) { j = 0; ++ch; tiles = as_entry_tiles(p, ch * 32, n, rows, G, lane, mine); }
            }
        };
        bool ok = true;
        while (f < f1 && ok) {
            seek();
            const AsEntry e = as_shfl(mine, j);
            const int per_head = __shfl_sync(0xffffffffu, tiles, j), n_rb = as_blocks(e.n_rows, rows);
            int kvh = (int)((f - at) / per_head), in = (int)((f - at) - (long long)kvh * per_head), rb = 0;
            for (int b0 = 0;; b0 += 32) {                    // the row block that has tile `in` of the head
                const int own = b0 + lane < n_rb ? as_count(p, e, b0 + lane, rows, G) : 0;
                int v = own;
                #pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += u; }
                const unsigned behind = __ballot_sync(0xffffffffu, v > in);
                if (behind) { const int k = __ffs(behind) - 1; rb = b0 + k; in -= __shfl_sync(0xffffffffu, v - own, k); break; }
                in -= __shfl_sync(0xffffffffu, v, 31);
            }
            const long long end_e = at + (long long)per_head * a.nkv;
            // units of the entry, one after the other
            for (; f < min(f1, end_e) && ok; in = 0) {
                const int r0 = rb * rows, r1 = min(r0 + rows, e.n_rows);
                const SpanTiles t = as_tiles(p, e, r0, r1, G);
                const int total = max(t.sink + t.near, 1);
                const long long u0 = f - in;
                int take = (int)min((long long)(total - in), f1 - f);
                if (!cut) take = in > 0 ? 0 : total;         // the unit is the CTA's where it begins
                if (take > 0) {
                    if (n_piece >= 2 && !mbar_wait_sleep_warp(&piece_empty[n_piece & 1], ((n_piece >> 1) - 1) & 1)) { ok = false; break; }
                    const int32_t* bt = a.block_table + (size_t)e.tab * a.pps;
                    if (lane == 0) {
                        AsPiece& x = pieces[n_piece & 1];
                        x.n_tiles = take; x.t0 = in; x.sink = t.sink; x.first = t.first; x.lo = t.lo; x.end = t.end; x.any = t.sink + t.near > 0;
                        const int p_first = e.cached + r0 / G, p_last = e.cached + (r1 - 1) / G;
                        x.all_hi = p.prefixes ? e.cached : min(max(p_first + 1, 0), a.pps * EXL3_PAGE);
                        x.all_lo = p.prefixes ? 0 : max(e.key_lo, a.window > p_last ? 0 : p_last - a.window + 1);
                        x.sinks = p.prefixes ? 0 : a.sinks;
                        x.tab = e.tab; x.row_base = e.row_base; x.r0 = r0; x.n_valid = r1 - r0; x.cached = e.cached; x.key_lo = e.key_lo; x.kvh = kvh;
                        x.ring = it;
                        x.c0 = (int)(u0 / share); x.index = cut ? (int)blockIdx.x - x.c0 : 0; x.count = cut ? (int)((u0 + total - 1) / share) - x.c0 + 1 : 1;
                        x.group = e.group;
                        mbar_arrive(&piece_full[n_piece & 1]);
                    }
                    // Q, when the scores of the piece before are computed: two copies, one per half of the head
                    if (n_piece > 0 && !mbar_wait_sleep_warp(q_empty, (n_piece - 1) & 1)) { ok = false; break; }
                    if (lane == 0) {
                        mbar_expect_tx(q_full, rows * 256);
                        for (int h = 0; h < 2; ++h) tma_load_4d(smem + h * Cfg::QHALF, &qmap, 0, h, kvh * G, e.row_base + r0 / G, q_full);
                    }
                    ++n_q;
                    ++n_piece;
                    for (int k = in; k < in + take && ok; ++k) {
                        const int kt = k < t.sink ? k : t.first + (k - t.sink);
                        int page = t.sink + t.near > 0 ? bt[kt >> 1] : -1;
                        if (page < 0 || page >= a.pages) page = a.pages;            // outside the pool: zeros, which the softmax threads mask
                        #pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            const int slot = it % SLOTS;
                            if (it >= SLOTS && !mbar_wait_sleep_warp(&kv_empty[slot], ((it / SLOTS) - 1) & 1)) { ok = false; break; }
                            if (lane == 0) {
                                mbar_expect_tx(&kv_full[slot], AS_TILE);
                                tma_load_5d(smem + Cfg::OFF_KV + slot * AS_TILE, v ? &vmap : &kmap, 0, (kt * AS_TK) & (EXL3_PAGE - 1), 0, kvh, page, &kv_full[slot]);
                            }
                            ++it;
                        }
                    }
                }
                f = u0 + (take > 0 ? in + take : total);
                if (++rb == n_rb) { rb = 0; ++kvh; }
            }
        }
        if (ok && n_piece >= 2 && !mbar_wait_sleep_warp(&piece_empty[n_piece & 1], ((n_piece >> 1) - 1) & 1)) ok = false;
        if (ok && lane == 0) { pieces[n_piece & 1].n_tiles = 0; mbar_arrive(&piece_full[n_piece & 1]); }
        failed = !ok;
        // not out before every copy has landed, whatever became of those who take them
        for (int i = max(0, it - SLOTS); i < it; ++i) mbar_wait_sleep_warp(&kv_full[i % SLOTS], (i / SLOTS) & 1);
        if (n_q > 0) mbar_wait_sleep_warp(q_full, (n_q - 1) & 1);
    } else if (warp == SW + 1) {
        // ===== MMA issuer: warp-uniform values, one elected lane
        const bool leader = elect_one();
        constexpr uint32_t HI = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);         // SBO, version 1, SWIZZLE_128B
        constexpr uint32_t LBO_K = 1u << 16, LBO_V = (uint32_t)((AS_TILE / 2) >> 4) << 16;
        auto mk = [](uint32_t lo, uint32_t hi) { return ((uint64_t)hi << 32) | lo; };
        const uint32_t q_lo = (smem_u32(smem) >> 4) | LBO_K, kv_lo = smem_u32(smem + Cfg::OFF_KV) >> 4;
        int done[2] = {0, 0};                                                             // tiles of each block
        for (int n_piece = 0; !failed; ++n_piece) {
            if (!mbar_wait_sleep_warp(&piece_full[n_piece & 1], (n_piece >> 1) & 1)) { failed = true; break; }
            const AsPiece& x = pieces[n_piece & 1];
            const int n_tiles = x.n_tiles, n_blocks = NB == 1 || x.n_valid <= AS_BLOCK ? 1 : 2, ring = x.ring;
            __syncwarp();
            if (lane == 0) mbar_arrive(&piece_empty[n_piece & 1]);
            if (n_tiles == 0) break;
            // S of block b from the K tile that is ring item `item`
            auto scores = [&](int b, int item, bool last) -> bool {
                const int slot = item % SLOTS;
                if (b == 0 && !mbar_wait_sleep_warp(&kv_full[slot], (item / SLOTS) & 1)) return false;
                tc_fence_after();
                if (leader) {
                    const uint32_t qb = q_lo + b * (AS_BLOCK * 128 >> 4), kb = (kv_lo + slot * (AS_TILE >> 4)) | LBO_K;
                    #pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t in = (kk & 3) * 32;
                        tc_mma_f16(tmem + b * 256, mk(qb + (((kk >> 2) * Cfg::QHALF + in) >> 4), HI), mk(kb + (((kk >> 2) * (AS_TILE / 2) + in) >> 4), HI),
                                   ATC_IDESC_S, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(&s_full[b]);
                    if (b == n_blocks - 1) { tc_commit(&kv_empty[slot]); if (last) tc_commit(q_empty); }
                }
                __syncwarp();
                return true;
            };
            if (!mbar_wait_warp(q_full, n_piece & 1)) { failed = true; break; }
            for (int b = 0; b < n_blocks && !failed; ++b)
                if (!scores(b, ring, n_tiles == 1)) failed = true;
            for (int j = 0; j < n_tiles && !failed; ++j) {
                const int item = ring + 2 * j + 1, slot = item % SLOTS;
                for (int b = 0; b < n_blocks && !failed; ++b) {
                    if (b == 0 && !mbar_wait_sleep_warp(&kv_full[slot], (item / SLOTS) & 1)) { failed = true; break; }
                    const uint32_t vb = (kv_lo + slot * (AS_TILE >> 4)) | LBO_V, tb = tmem + b * 256;
                    #pragma unroll
                    for (int half_ = 0; half_ < 2 && !failed; ++half_) {
                        if (!mbar_wait_warp(half_ ? &p_full[b] : &p_half[b], done[b] & 1)) { failed = true; break; }
                        tc_fence_after();
                        if (leader) {
                            #pragma unroll
                            for (int kk = 4 * half_; kk < 4 * half_ + 4; ++kk)
                                tc_mma_f16_ts(tb + 128, tb + kk * 8, mk(vb + kk * (2048 >> 4), HI), ATC_IDESC_PV, (j > 0 || kk > 0) ? 1u : 0u);
                            if (half_ && b == n_blocks - 1) tc_commit(&kv_empty[slot]);
                        }
                        __syncwarp();
                    }
                    ++done[b];
                    if (failed) break;
                    // S of the next tile over P of this one: the tensor core runs the product before it first
                    if (j + 1 < n_tiles) { if (!scores(b, item + 1, j + 2 == n_tiles)) failed = true; }
                    else { if (leader) tc_commit(&o_full[b]); __syncwarp(); }
                }
            }
        }
    } else {
        // ===== softmax: thread = row
        const int blk = warp >> 2, r = tid - blk * AS_BLOCK;
        const uint32_t ts = tmem + blk * 256 + ((uint32_t)((warp & 3) * 32) << 16), to_ = ts + 128;
        const float scale = a.scale_log2;
        uint8_t* stage = smem + Cfg::OFF_STAGE + warp * 2048;
        int done = 0, begun = 0;                                            // tiles and pieces of this block
        const int per8 = 8 / G, left8 = 8 - per8 * G;                       // rows and heads that 8 packed rows go on
        for (int n_piece = 0; !failed; ++n_piece) {
            if (!mbar_wait_warp(&piece_full[n_piece & 1], (n_piece >> 1) & 1)) { failed = true; break; }
            const AsPiece x = pieces[n_piece & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(&piece_empty[n_piece & 1]);
            if (x.n_tiles == 0) break;
            if (blk * AS_BLOCK >= x.n_valid) continue;
            int lo = 0, hi = 0;
            if (tid < x.n_valid) {
                if (p.prefixes) hi = x.cached;
                else {
                    const int pos = x.cached + (x.r0 + tid) / G;
                    hi = min(max(pos + 1, 0), a.pps * EXL3_PAGE);
                    lo = max(x.key_lo, a.window > pos ? 0 : pos - a.window + 1);
                }
            }
            const int32_t* bt = a.block_table + (size_t)x.tab * a.pps;
            auto key_tile = [&](int j) -> int { const int i = x.t0 + j; return i < x.sink ? i : x.first + (i - x.sink); };
            // a tile's page is read a tile ahead and looked at where it counts: a comparison behind the load waits for it (860 cycles per tile)
            int page = x.any ? bt[key_tile(0) >> 1] : -1;
            // m_used: the exponents' reference; r_true: the maximum before the scale, which is positive
            float m_used = -INFINITY, r_true = -INFINITY, l = 0.f;
            bool far = false;                                               // of the warp, from some tile on
            for (int j = 0; j < x.n_tiles; ++j, ++done) {
                const int kb = key_tile(j) * AS_TK;
                const bool gone = page < 0 || page >= a.pages;
                if (j + 1 < x.n_tiles) page = bt[key_tile(j + 1) >> 1];
                if (!mbar_wait_warp(&s_full[blk], done & 1)) { failed = true; break; }
                tc_fence_after();
                // 32 scores at a time: the last two chunks are read twice, once for the maximum and again while the first ones are in work
                // (all 128 held through both passes take 230 registers)
                float x0[32], x1[32], x2[32];
                auto chunk_at = [&](int c, float (&v)[32]) { tc_ld32(ts + c * 32, v); };
                const bool clear = !gone && kb + AS_TK <= x.all_hi && (kb >= x.all_lo || kb + AS_TK <= x.sinks);
                auto mask = [&](int c, float (&v)[32]) {
                    if (!clear) {                            // keys that the row sees, as bits: a predicate per key and no comparisons
                        auto below = [](int n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; };
                        const int k0 = kb + c * 32;
                        const uint32_t see = gone ? 0u : below(hi - k0) & (~below(lo - k0) | below(x.sinks - k0));
                        #pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = see >> i & 1 ? v[i] : -INFINITY;
                    }
                };
                float mx0 = -INFINITY, mx1 = -INFINITY;
                auto maximum = [&](const float (&v)[32]) {
                    #pragma unroll
                    for (int i = 0; i < 32; i += 4) { mx0 = fmax3(mx0, v[i], v[i + 1]); mx1 = fmax3(mx1, v[i + 2], v[i + 3]); }
                };
                // values that no row of the unit sees may be anything (0 * NaN would spoil O): cleared by the first block, whose product
                // comes first, a key per thread
                auto clear_values = [&]() -> bool {
                    if (blk != 0 || gone || (kb + AS_TK <= x.end && (kb >= x.lo || kb + AS_TK <= x.sinks))) return true;
                    const int item = x.ring + 2 * j + 1, slot = item % SLOTS;
                    if (!mbar_wait_sleep_warp(&kv_full[slot], (item / SLOTS) & 1)) return false;
                    const int key = kb + r;
                    if (!(key < x.end && (key >= x.lo || key < x.sinks))) {
                        #pragma unroll
                        for (int c = 0; c < 16; ++c)
                            *reinterpret_cast<uint4*>(smem + Cfg::OFF_KV + slot * AS_TILE + (c >> 3) * (AS_TILE / 2) + r * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                    return true;
                };
                auto announce = [&](uint64_t* bar) {
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar);
                };
                auto rescale_o = [&](float corr) {                          // O holds the tiles before: the scores came after their product
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        tc_ld32(to_ + c * 32, x1);
                        tc_wait_ld();
                        #pragma unroll
                        for (int i = 0; i < 32; ++i) x1[i] *= corr;
                        tc_st32(to_ + c * 32, x1);
                    }
                };
                float2 sum = make_float2(0.f, 0.f);
                const bool entered = !far;
                if (!far) {
                    chunk_at(2, x0); chunk_at(3, x1); chunk_at(0, x2);
                    tc_wait_ld();
                    mask(2, x0); maximum(x0);
                    chunk_at(1, x0);
                    mask(3, x1); maximum(x1);
                    mask(0, x2); maximum(x2);
                    tc_wait_ld();
                    mask(1, x0); maximum(x0);
                    r_true = fmaxf(r_true, fmaxf(mx0, mx1));
                    const float m_true = __fmul_rn(r_true, scale);
                    // the reference moves only when the maximum has grown by 2^8, so O is seldom rescaled
                    const bool move = m_true > m_used + ATC_RESCALE_THRESHOLD || (m_used == -INFINITY && m_true > -INFINITY);
                    float corr = 1.0f;
                    if (__any_sync(0xffffffffu, move)) {
                        far = __any_sync(0xffffffffu, move && hi > 0 && fabsf(m_true) >= AS_FAR);     // rows behind the unit's last may hold anything
                        if (!far) {
                            const bool rescale = move && m_used != -INFINITY;
                            if (rescale) corr = ex2_approx(m_used - m_true);
                            if (move) m_used = m_true;
                            if (__any_sync(0xffffffffu, rescale)) rescale_o(corr);
                        }
                    }
                    if (!far) {
                        if (!clear_values()) { failed = true; break; }
                        const float nref = m_used == -INFINITY ? 0.f : -m_used;
                        const float2 scale2 = make_float2(scale, scale), nref2 = make_float2(nref, nref);
                        uint32_t w[32];
                        auto weights = [&](const float (&v)[32], int at) {
                            #pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 y = fma2(make_float2(v[i], v[i + 1]), scale2, nref2);
                                const float2 ex = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                                sum = add2(sum, ex);
                                w[at + (i >> 1)] = pack_h2(ex.x, ex.y);             // the one rounding of a weight, as the product takes it
                            }
                        };
                        chunk_at(2, x1);
                        weights(x2, 0);
                        weights(x0, 16);
                        tc_st32u(ts, w);
                        tc_wait_ld();
                        announce(&p_half[blk]);
                        chunk_at(3, x0);
                        mask(2, x1);
                        weights(x1, 0);
                        tc_wait_ld();
                        mask(3, x0);
                        weights(x0, 16);
                        tc_st32u(ts + 32, w);
                        announce(&p_full[blk]);
                        l = l * corr + (sum.x + sum.y);
                        continue;
                    }
                }
                // A reference far from 0, in this tile or one before: 32 scores at a time, and the reference is always the maximum.  (A way of its own to
                // the end of the tile; within the other one it took 2 % more of every call.)
                const float r_before = r_true;
                #pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    chunk_at(c, x0);
                    tc_wait_ld();
                    mask(c, x0);
                    maximum(x0);
                }
                r_true = fmaxf(r_true, fmaxf(mx0, mx1));
                const float m_true = __fmul_rn(r_true, scale), grown = entered ? m_used - m_true : (r_before - r_true) * scale;
                const float corr = m_used != -INFINITY && grown < 0.f ? ex2_approx(grown) : 1.0f, origin = r_true == -INFINITY ? 0.f : r_true;
                m_used = m_true;
                if (__any_sync(0xffffffffu, corr != 1.0f)) rescale_o(corr);
                if (!clear_values()) { failed = true; break; }
                #pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    chunk_at(c, x0);
                    tc_wait_ld();
                    mask(c, x0);
                    uint32_t w[16];
                    #pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 ex = make_float2(ex2_approx((x0[i] - origin) * scale), ex2_approx((x0[i + 1] - origin) * scale));
                        sum = add2(sum, ex);
                        w[i >> 1] = pack_h2(ex.x, ex.y);
                    }
                    tc_st16u(ts + c * 16, w);                               // over scores that are read already
                    if (c & 1) announce(c == 1 ? &p_half[blk] : &p_full[blk]);
                }
                l = l * corr + (sum.x + sum.y);
            }
            failed = __any_sync(0xffffffffu, failed);
            if (failed) break;
            // ===== O -> output or partial sum, some columns at a time by way of shared memory: rows of 64 bytes, eight per instruction
            if (!mbar_wait_warp(&o_full[blk], begun & 1)) { failed = true; break; }
            ++begun;
            tc_fence_after();
            const int n_mine = min(32, x.n_valid - warp * 32);
            const bool direct = !p.prefixes && x.count == 1 && x.group < 0;
            auto row_of = [&](int i) -> size_t {                            // (row, head) of the warp's row i
                const int pk = x.r0 + warp * 32 + i, q = pk / G;
                return (size_t)(x.row_base + q) * a.nq + x.kvh * G + (pk - q * G);
            };
            // Partial sums that span_join_kernel reads go by row, [row][head][SPAN_PART] (of a prefix [place] in front); those of a cut own span to
            // the CTA's place for its first or last unit, as the threads have them: [warp][4 dims][lane], then a warp's maxima and sums.
            float* by_row = p.prefixes ? p.partial + (size_t)x.index * a.rows * a.nq * SPAN_PART : p.rest;
            auto own_part = [&](int index) -> float* {
                return p.partial + ((size_t)(2 * (x.c0 + index) + (index == 0 ? 1 : 0)) * SW + warp) * 32 * SPAN_PART;
            };
            const int sr = lane >> 2, sc = lane & 3;
            // 32 columns of the warp's rows in fp16, or 16 in fp32, by way of shared memory: rows of 64 bytes, eight per instruction
            size_t at[4];                                                   // of rows sr, 8 + sr, ..
            {
                const int pk = x.r0 + warp * 32 + sr;
                int q = pk / G, g0 = pk - q * G;
                #pragma unroll
                for (int g = 0; g < 4; ++g) {
                    at[g] = (size_t)(x.row_base + q) * a.nq + x.kvh * G + g0;
                    q += per8; g0 += left8;
                    if (g0 >= G) { g0 -= G; ++q; }
                }
            }
            auto put = [&](const uint4 (&v)[4], auto store) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = v[i];
                __syncwarp();
                #pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int i = 8 * g + sr;
                    if (i < n_mine) store(g, *reinterpret_cast<const uint4*>(stage + i * 64 + ((sc ^ ((i >> 1) & 3)) << 4)));
                }
                __syncwarp();
            };
            auto put_half = [&](const float (&o)[32], float inv, int c) {   // columns 32 c .. of the output
                uint4 v[4];
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = make_uint4(pack_h2(o[8 * i] * inv, o[8 * i + 1] * inv), pack_h2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                      pack_h2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack_h2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                put(v, [&](int g, uint4 y) { *reinterpret_cast<uint4*>(a.o + at[g] * 128 + c * 32 + sc * 8) = y; });
            };
            auto put_float = [&](const float (&o)[32], int c) {             // columns 32 c .. of a partial sum by row
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4 v[4];
                    #pragma unroll
                    for (int i = 0; i < 4; ++i)
                        v[i] = make_uint4(__float_as_uint(o[16 * h + 4 * i]), __float_as_uint(o[16 * h + 4 * i + 1]),
                                          __float_as_uint(o[16 * h + 4 * i + 2]), __float_as_uint(o[16 * h + 4 * i + 3]));
                    put(v, [&](int g, uint4 y) { *reinterpret_cast<uint4*>(by_row + at[g] * SPAN_PART + c * 32 + h * 16 + sc * 4) = y; });
                }
            };
            const bool own = !p.prefixes && x.count > 1;
            float* mine = own ? own_part(x.index) : nullptr;
            const float inv = l > 0.f ? 1.0f / l : 0.f;
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                float o[32];
                tc_ld32(to_ + c * 32, o);
                tc_wait_ld();
                if (direct) put_half(o, inv, c);
                else if (own) {
                    #pragma unroll
                    for (int i = 0; i < 8; ++i)
                        reinterpret_cast<float4*>(mine)[(c * 8 + i) * 32 + lane] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                } else put_float(o, c);
            }
            if (direct) continue;
            if (!own) {
                if (lane < n_mine) {
                    const size_t me = row_of(lane) * SPAN_PART + 128;
                    *reinterpret_cast<float2*>(by_row + me) = make_float2(m_used, l);
                    // a prefix's places are read up to the most parts that a unit of its length can have
                    if (p.prefixes && x.index == x.count - 1 && cut)
                        for (int k = x.count; k < span_places((x.cached + AS_TK - 1) / AS_TK, (int)share); ++k)
                            *reinterpret_cast<float2*>(p.partial + (size_t)k * a.rows * a.nq * SPAN_PART + me) = make_float2(-INFINITY, 0.f);
                }
                continue;
            }
            reinterpret_cast<float2*>(mine + 32 * 128)[lane] = make_float2(m_used, l);
            __threadfence();
            __syncwarp();
            int before = 0;
            if (lane == 0) {
                before = atomicAdd(p.counters + x.c0 * SW + warp, 1);
                if (before == x.count - 1) p.counters[x.c0 * SW + warp] = 0;
            }
            if (__shfl_sync(0xffffffffu, before, 0) != x.count - 1) continue;
            __threadfence();
            // all parts of the unit are there: a thread per row.  Of two, this one's is still in tensor memory, and the other one's values are asked for
            // 32 columns ahead; each product is rounded before the sum, so that it does not matter which of the two is here.
            if (x.count == 2) {
                const float* other = own_part(1 - x.index);
                float4 v[8];
                auto fetch = [&](int c) {
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = __ldcg(reinterpret_cast<const float4*>(other) + (c * 8 + i) * 32 + lane);
                };
                const float2 y = __ldcg(reinterpret_cast<const float2*>(other + 32 * 128) + lane);
                fetch(0);
                const float top2 = fmaxf(m_used, y.x), ref2 = top2 == -INFINITY ? 0.f : top2;
                const float w0 = exp2f(m_used - ref2), w1 = exp2f(y.x - ref2), l2 = __fadd_rn(__fmul_rn(l, w0), __fmul_rn(y.y, w1));
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float o[32];
                    tc_ld32(to_ + c * 32, o);
                    tc_wait_ld();
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        o[4 * i] = __fadd_rn(__fmul_rn(o[4 * i], w0), __fmul_rn(v[i].x, w1));
                        o[4 * i + 1] = __fadd_rn(__fmul_rn(o[4 * i + 1], w0), __fmul_rn(v[i].y, w1));
                        o[4 * i + 2] = __fadd_rn(__fmul_rn(o[4 * i + 2], w0), __fmul_rn(v[i].z, w1));
                        o[4 * i + 3] = __fadd_rn(__fmul_rn(o[4 * i + 3], w0), __fmul_rn(v[i].w, w1));
                    }
                    if (c < 3) fetch(c + 1);
                    if (x.group < 0) put_half(o, l2 > 0.f ? 1.0f / l2 : 0.f, c);
                    else put_float(o, c);
                }
                if (x.group >= 0 && lane < n_mine) *reinterpret_cast<float2*>(by_row + row_of(lane) * SPAN_PART + 128) = make_float2(top2, l2);
                continue;
            }
            auto max_sum = [&](int k) -> float2 { return __ldcg(reinterpret_cast<const float2*>(own_part(k) + 32 * 128) + lane); };
            float top = -INFINITY, l_all = 0.f;
            #pragma unroll 4
            for (int k = 0; k < x.count; ++k) top = fmaxf(top, max_sum(k).x);
            const float ref = top == -INFINITY ? 0.f : top;
            for (int c = 0; c < 4; ++c) {
                float o[32];
                #pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.f;
                #pragma unroll 2
                for (int k = 0; k < x.count; ++k) {
                    const float2 y = max_sum(k);
                    float4 v[8];
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = __ldcg(reinterpret_cast<const float4*>(own_part(k)) + (c * 8 + i) * 32 + lane);
                    const float w = exp2f(y.x - ref);
                    if (c == 0) l_all = fmaf(y.y, w, l_all);
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        o[4 * i] = fmaf(v[i].x, w, o[4 * i]); o[4 * i + 1] = fmaf(v[i].y, w, o[4 * i + 1]);
                        o[4 * i + 2] = fmaf(v[i].z, w, o[4 * i + 2]); o[4 * i + 3] = fmaf(v[i].w, w, o[4 * i + 3]);
                    }
                }
                __syncwarp();
                if (x.group < 0) put_half(o, l_all > 0.f ? 1.0f / l_all : 0.f, c);
                else put_float(o, c);
            }
            if (x.group >= 0 && lane < n_mine) *reinterpret_cast<float2*>(by_row + row_of(lane) * SPAN_PART + 128) = make_float2(top, l_all);
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
}

// Adds the partial sums of its prefix to every row of a sequence that has one: a warp takes U (row, head) pairs, four where there are many,
// and one where one each leaves SMs idle: then what counts is how often a warp waits for memory.
struct SpanJoinParams { SpanArgs a; const float* prefix; const int* share; const float* rest; };
template <int U>
__global__ void __launch_bounds__(256) span_join_kernel(const SpanJoinParams p)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const SpanArgs& a = p.a;
    const int lane = threadIdx.x & 31;
    const long long n = (long long)a.rows * a.nq, w0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * U;
    if (w0 >= n) { pdl_wait(); return; }
    const int row = (int)(w0 / a.nq);                        // lengths and groups were there before the call began
    // a row's group and prefix; U pairs belong to one row where the head count allows it
    int len[U];
    bool any = false;
    int last_row = -1, last_len = 0;
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        len[u] = 0;
        if (w0 + u >= n) continue;
        const int r = u == 0 ? row : (int)((w0 + u) / a.nq);
        if (r != last_row) {
            int b;
            if (a.cu_q) {
                int lo = 0, hi = a.bsz;
                while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.cu_q[mid] <= r) lo = mid; else hi = mid; }
                b = lo;
            } else b = r / a.q_len;
            const SpanSeq s = span_seq(a, b);
            last_row = r;
            last_len = r < s.row_base || r >= s.row_base + s.ql ? 0 : span_group(a, b, s.cached).len;
        }
        len[u] = last_len;
        any |= last_len > 0;
    }
    pdl_wait();
    if (!any) return;
    const int share = *p.share;
    int places = 0;
    #pragma unroll
    for (int u = 0; u < U; ++u) if (len[u]) places = max(places, span_places((len[u] + AS_TK - 1) / AS_TK, share));
    SpanSum sum[U];
    // place 0 of the sum is the sequence's own part; a place behind a shorter prefix's last stands for that one with weight 0
    span_merge<U == 1 ? 12 : 4>(sum, places + 1, [&](int k, int u) -> const float* {
        const long long at = min(w0 + u, n - 1);
        return k == 0 ? p.rest + at * SPAN_PART : p.prefix + ((size_t)(k - 1) * n + at) * SPAN_PART;
    }, [&](int k, int u) -> bool { return k == 0 || k - 1 < (len[u] ? span_places((len[u] + AS_TK - 1) / AS_TK, share) : 0); }, lane);
    #pragma unroll
    for (int u = 0; u < U; ++u)
        if (len[u]) reinterpret_cast<uint2*>(a.o)[(w0 + u) * 32 + lane] = span_result(sum[u]);
}

}  // namespace exl3
