// What the attention over spans of the cache shares: which keys a sequence's rows see, and where they stand.
//
//   o[row, h] = sum_j w_j v[j] / sum_j w_j,   w_j = exp(scale * q[row, h] . k[j, h / G]),   j over the keys that the row sees
//   window: j <= p and (j > p - window or j < sinks);   shared prefix: j <= p;   p = cached tokens + number of the row in its sequence
//
// A row whose span is empty gives zeros.  Keys of a block-table entry outside the pool are left out, and entries without a visible key are
// not read.
#pragma once
#include "common.cuh"

namespace exl3 {

struct SpanArgs {
    const half* q; half* o;                       // [rows, nq, 128]
    const half* kc; const half* vc;               // [pages, 256, nkv, 128]
    const int32_t* block_table;                   // [bsz, pps]
    const int32_t* seqlens;                       // [bsz] cached tokens in front of a sequence's rows
    const int32_t* cu_q;                          // [bsz + 1], or NULL: q_len rows each
    const int32_t* group_start;                   // [n_groups + 1] first sequence of every group (shared prefixes), or NULL
    const int32_t* prefix_lens;                   // [n_groups]
    int bsz, q_len, rows, nq, nkv, pages, pps, n_groups;
    int window, sinks;                            // window: INT_MAX without one
    float scale_log2;
    int beside;                                   // SMs that the kernels of few and of many rows share, running beside one another; 0: each has the GPU
    int unit_rows;                                // then: packed rows of a unit of the tcgen05 kernel
};

constexpr int SPAN_MAX_LEN = 1 << 30;
// 1/20 us that an SM takes per kv head: for a tile of 128 keys and a few rows (64 KB at 55 GB/s), for one and 256 packed rows, and for a unit of 256 rows
// besides; units of 128, two at a time, take 4/5.  Fitted to 12 batches at 23 splits of the SMs each: 0 to 9 % above the best of the 23, where the
// classes in calls of their own take 3 to 44 % more than that.
constexpr int SPAN_FEW_TILE = 24, SPAN_MANY_TILE = 46, SPAN_MANY_UNIT = 120;

// A sequence's place in the call.  ql 0: it has no rows, more than the call declared, or rows that the call does not have.
struct SpanSeq { int row_base, ql, cached; };
__device__ __forceinline__ SpanSeq span_seq(const SpanArgs& a, int b)
{
    SpanSeq s;
    s.row_base = a.cu_q ? a.cu_q[b] : b * a.q_len;
    s.ql = a.cu_q ? a.cu_q[b + 1] - s.row_base : a.q_len;
    if (s.ql < 0 || s.ql > a.q_len || s.row_base < 0 || s.row_base > a.rows - s.ql) s.ql = 0;
    s.cached = max(min(a.seqlens[b], SPAN_MAX_LEN), -SPAN_MAX_LEN);
    return s;
}

// The group of a sequence: its first sequence, whose table has the prefix, and the prefix's tokens.  A sequence of no group, or one that
// has not cached the whole prefix, has none and is computed on its own.
struct SpanGroup { int g, first, len; };
__device__ __forceinline__ SpanGroup span_group(const SpanArgs& a, int b, int cached)
{
    SpanGroup r = {-1, b, 0};
    if (a.n_groups == 0) return r;
    int lo = 0, hi = a.n_groups;                  // group_start[lo] <= b < group_start[hi]
    int from = a.group_start[0], len = a.prefix_lens[0];        // asked for together with the end: one group is the common case
    if (from > b || a.group_start[hi] <= b) return r;
    if (hi > 1) {
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.group_start[mid] <= b) lo = mid; else hi = mid; }
        from = a.group_start[lo]; len = a.prefix_lens[lo];
    }
    len = min(len, a.pps * EXL3_PAGE);
    if (len <= 0 || len > cached) return r;
    r.g = lo; r.first = max(from, 0); r.len = len;
    return r;
}

}  // namespace exl3

namespace exl3 {

// The key tiles that a run of rows at positions p_first..p_last sees: `sink` tiles from 0 on, then tiles first .. first + near - 1.  Keys in
// front of key_lo are not part of it.
struct SpanTiles { int sink, first, near, lo, end; };
template <int TK>
__device__ __forceinline__ SpanTiles span_tiles(const SpanArgs& a, int p_first, int p_last, int key_lo)
{
    SpanTiles t;
    t.end = min(max(p_last + 1, 0), a.pps * EXL3_PAGE);
    t.lo = max(key_lo, a.window > p_first ? 0 : p_first - a.window + 1);
    t.first = t.lo / TK;
    t.near = t.end > t.lo ? (t.end + TK - 1) / TK - t.first : 0;
    t.sink = (min(a.sinks, t.end) + TK - 1) / TK;
    if (t.near > 0) t.sink = min(t.sink, t.first);
    return t;
}

// Where both kernels run beside one another, their split of the SMs goes by the time of an SM that either class needs, as the lengths have it: whole
// numbers, so that every CTA of both kernels finds the same.  The load of sequence b (a tenth of a second at most):
struct SpanLoad { unsigned few, many; };
__device__ __forceinline__ void span_load(const SpanArgs& a, int b, int few_rows, SpanLoad& load)
{
    const int G = a.nq / a.nkv;
    const SpanSeq s = span_seq(a, b);
    if (s.ql == 0) return;
    const int last = s.cached + s.ql - 1, packed = s.ql * G;
    constexpr unsigned MOST = 1u << 21;                 // of 1024 sequences together 2^31
    if (packed <= few_rows) {
        const SpanTiles t = span_tiles<64>(a, s.cached, last, 0);
        load.few += min((unsigned)max(t.sink + t.near, 1), MOST / SPAN_FEW_TILE) * (SPAN_FEW_TILE / 2);
    } else {                                            // its units' tiles: halfway between the first's and the last's
        const int step = a.unit_rows / G;
        const SpanTiles t0 = span_tiles<128>(a, s.cached, min(s.cached + step - 1, last), 0), t1 = span_tiles<128>(a, max(last - step + 1, s.cached), last, 0);
        const unsigned unit = min((unsigned)(t0.sink + t0.near + t1.sink + t1.near), MOST / SPAN_MANY_TILE) * (SPAN_MANY_TILE / 2) + SPAN_MANY_UNIT;
        load.many += min((unsigned)((packed + a.unit_rows - 1) / a.unit_rows), MOST / unit) * unit;
    }
}
// a warp's part of the loads, to shared memory
__device__ __forceinline__ void span_load_put(SpanLoad* loads, int warp, const SpanLoad& load, int lane)
{
    const unsigned few = __reduce_add_sync(0xffffffffu, load.few), many = __reduce_add_sync(0xffffffffu, load.many);
    if (lane == 0) loads[warp] = {few, many};
}
// the SMs of the kernel for few rows
__device__ __forceinline__ int span_few_sms(const SpanArgs& a, const SpanLoad* loads, int warps)
{
    unsigned few = 0, many = 0;
    for (int w = 0; w < warps; ++w) { few += loads[w].few; many += loads[w].many; }
    if (a.unit_rows <= 128) many -= many / 5;
    if (few == 0 || many == 0) return few ? a.beside : 0;
    return min(max((int)__fdiv_rn(__fmul_rn((float)a.beside, (float)few), __fadd_rn((float)few, (float)many)), 4), a.beside - 4);
}

// Partial sums of a row and head: 128 dims, the exponents' reference, the sum of the weights
constexpr int SPAN_PART = 132;
constexpr int AS_TK = 128;                               // key tile of the tcgen05 kernel, in which splits of a prefix are counted
// Partial sums that a unit of so many tiles can have where CTAs take `share` tiles each; 0: units are not cut
__device__ __forceinline__ int span_places(int tiles, int share) { return share > 0 ? (tiles - 1) / share + 2 : 1; }

// Sums of U rows over n parts each.  A warp; lane = four dims, all lanes have top and l.  part(k, u): part k of row u,
// there(k, u): whether the row has it.  What waits for memory
// is asked for together: the maxima and sums of all parts, and the values of AHEAD parts of every row, whatever the maxima are (a part
// without keys, or a place that nobody wrote values to, has weight 0 and is not looked at).  One after the other, 4 us per row.
struct SpanSum { float4 acc; float top, l; };
template <int AHEAD, int U, typename Part, typename There>
__device__ __forceinline__ void span_merge(SpanSum (&s)[U], int n, Part part, There there, int lane)
{
    #pragma unroll
    for (int u = 0; u < U; ++u) s[u] = {make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f};
    for (int k0 = 0; k0 < n; k0 += 32) {
        const int cnt = min(32, n - k0);
        float2 x[U];
        float4 v[AHEAD][U];
        auto fetch = [&](int k) {
            #pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                #pragma unroll
                for (int u = 0; u < U; ++u) v[i][u] = __ldcg(reinterpret_cast<const float4*>(part(k0 + min(k + i, cnt - 1), u)) + lane);
        };
        #pragma unroll
        for (int u = 0; u < U; ++u) x[u] = __ldcg(reinterpret_cast<const float2*>(part(k0 + min(lane, cnt - 1), u) + 128));
        fetch(0);
        float w[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            if (lane >= cnt || !there(k0 + lane, u)) x[u] = make_float2(-INFINITY, 0.f);
            float top = x[u].x;
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(top, s[u].top);
            w[u] = x[u].x == -INFINITY ? 0.f : exp2f(x[u].x - top);
            float l = x[u].y * w[u];
            if (x[u].x == -INFINITY) l = 0.f;
            #pragma unroll
            for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const float c = s[u].top == -INFINITY ? 0.f : exp2f(s[u].top - top);
            s[u].acc.x *= c; s[u].acc.y *= c; s[u].acc.z *= c; s[u].acc.w *= c;
            s[u].l = s[u].l * c + l;
            s[u].top = top;
        }
        for (int k = 0; k < cnt; k += AHEAD) {
            #pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                #pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float wk = __shfl_sync(0xffffffffu, w[u], min(k + i, 31));
                    if (k + i < cnt && wk != 0.f) {
                        s[u].acc.x = fmaf(v[i][u].x, wk, s[u].acc.x); s[u].acc.y = fmaf(v[i][u].y, wk, s[u].acc.y);
                        s[u].acc.z = fmaf(v[i][u].z, wk, s[u].acc.z); s[u].acc.w = fmaf(v[i][u].w, wk, s[u].acc.w);
                    }
                }
            if (k + AHEAD < cnt) fetch(k + AHEAD);
        }
    }
}
__device__ __forceinline__ uint2 span_result(const SpanSum& s)
{
    const float inv = s.l > 0.f ? 1.0f / s.l : 0.f;
    const half2 a = __floats2half2_rn(s.acc.x * inv, s.acc.y * inv), b = __floats2half2_rn(s.acc.z * inv, s.acc.w * inv);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// A (row, head)'s finished sum: to the output, or to where span_join_kernel adds the prefix.  A warp, lane = four dims.
__device__ __forceinline__ void span_put(const SpanArgs& a, float* rest, int group, size_t at, const SpanSum& s, int lane)
{
    if (group < 0) { reinterpret_cast<uint2*>(a.o)[at * 32 + lane] = span_result(s); return; }
    reinterpret_cast<float4*>(rest + at * SPAN_PART)[lane] = s.acc;
    if (lane == 0) *reinterpret_cast<float2*>(rest + at * SPAN_PART + 128) = make_float2(s.top, s.l);
}

}  // namespace exl3
