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
};

constexpr int SPAN_MAX_LEN = 1 << 30;

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
    int lo = 0, hi = a.n_groups;                  // group_start[lo] <= b
    if (a.group_start[0] > b || a.group_start[hi] <= b) return r;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.group_start[mid] <= b) lo = mid; else hi = mid; }
    const int len = min(a.prefix_lens[lo], a.pps * EXL3_PAGE);
    if (len <= 0 || len > cached) return r;
    r.g = lo; r.first = max(a.group_start[lo], 0); r.len = len;
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

// Partial sums of a row and head: 128 dims, the exponents' reference, the sum of the weights
constexpr int SPAN_PART = 132;
constexpr int AS_TK = 128;                               // key tile of the tcgen05 kernel, in which splits of a prefix are counted
__device__ __forceinline__ int as_splits(int tiles, int chunk) { return max(1, (tiles + chunk - 1) / chunk); }

// A row's sum, to which one part after the other is added.  Lane = four dims; all lanes have top and l.
struct AsSum { float4 acc; float top, l; };
__device__ __forceinline__ void as_add(AsSum& s, const float* part, int lane)
{
    const float4 v = __ldcg(reinterpret_cast<const float4*>(part) + lane);
    const float2 x = __ldcg(reinterpret_cast<const float2*>(part + 128));
    const float top = fmaxf(s.top, x.x);
    const float c0 = s.top == -INFINITY ? 0.f : exp2f(s.top - top), c1 = x.x == -INFINITY ? 0.f : exp2f(x.x - top);
    s.acc.x = s.acc.x * c0 + v.x * c1; s.acc.y = s.acc.y * c0 + v.y * c1; s.acc.z = s.acc.z * c0 + v.z * c1; s.acc.w = s.acc.w * c0 + v.w * c1;
    s.l = s.l * c0 + x.y * c1;
    s.top = top;
}

}  // namespace exl3
