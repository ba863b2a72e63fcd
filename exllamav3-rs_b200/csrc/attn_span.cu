// exl3_window_attn_paged and exl3_prefix_attn_paged: attention over spans of the paged cache.
#include <limits.h>
#include <math.h>
#include "attn_span.cuh"

namespace {

using namespace exl3;

// The plain kernel: a warp per (row, head), one key at a time, lane = 4 dims.
__global__ void __launch_bounds__(256) span_plain_kernel(const SpanArgs a, int early)
{
    pdl_enter_first(early);
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= (long long)a.rows * a.nq) return;
    const int row = (int)(w / a.nq), head = (int)(w % a.nq), kvh = head / (a.nq / a.nkv);
    int b = 0;
    if (a.cu_q) {
        int lo = 0, hi = a.bsz;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.cu_q[mid] <= row) lo = mid; else hi = mid; }
        b = lo;
    } else b = row / a.q_len;
    const SpanSeq s = span_seq(a, b);
    if (row < s.row_base || row >= s.row_base + s.ql) return;
    const int p = s.cached + (row - s.row_base), end = min(p + 1, a.pps * EXL3_PAGE);
    const SpanGroup g = span_group(a, b, s.cached);
    const uint2 qr = reinterpret_cast<const uint2*>(a.q + ((size_t)row * a.nq + head) * 128)[lane];
    const float2 q0 = __half22float2(*reinterpret_cast<const half2*>(&qr.x)), q1 = __half22float2(*reinterpret_cast<const half2*>(&qr.y));
    const int near = a.window > p ? 0 : p - a.window + 1;
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = a.sinks > 0 ? 0 : near; j < end; ++j) {
        if (j < near && j >= a.sinks) j = near;
        if (j >= end) break;
        const int page = a.block_table[(size_t)(j < g.len ? g.first : b) * a.pps + (j >> 8)];
        if (page < 0 || page >= a.pages) continue;
        const size_t at = (((size_t)page * EXL3_PAGE + (j & 255)) * a.nkv + kvh) * 32 + lane;
        const uint2 kr = reinterpret_cast<const uint2*>(a.kc)[at], vr = reinterpret_cast<const uint2*>(a.vc)[at];
        const float2 k0 = __half22float2(*reinterpret_cast<const half2*>(&kr.x)), k1 = __half22float2(*reinterpret_cast<const half2*>(&kr.y));
        const float2 v0 = __half22float2(*reinterpret_cast<const half2*>(&vr.x)), v1 = __half22float2(*reinterpret_cast<const half2*>(&vr.y));
        float x = q0.x * k0.x + q0.y * k0.y + q1.x * k1.x + q1.y * k1.y;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        x *= a.scale_log2;
        const float mn = fmaxf(m, x), c = m == -INFINITY ? 0.f : exp2f(m - mn), e = mn == -INFINITY ? 0.f : exp2f(x - mn);
        m = mn; l = l * c + e;
        acc[0] = acc[0] * c + e * v0.x; acc[1] = acc[1] * c + e * v0.y; acc[2] = acc[2] * c + e * v1.x; acc[3] = acc[3] * c + e * v1.y;
    }
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    const half2 o0 = __floats2half2_rn(acc[0] * inv, acc[1] * inv), o1 = __floats2half2_rn(acc[2] * inv, acc[3] * inv);
    reinterpret_cast<uint2*>(a.o + ((size_t)row * a.nq + head) * 128)[lane] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&o0), *reinterpret_cast<const uint32_t*>(&o1));
}

// a call without rows touches none of its tensors, whose pointers may be null then
bool span_empty(const SpanArgs& a) { return a.bsz == 0 || a.q_len == 0 || a.rows == 0; }

int span_check(exl3_ctx* ctx, const SpanArgs& a, int hd, float sm_scale, const char* what)
{
    char msg[128];
    auto bad = [&](int code, const char* why) { snprintf(msg, sizeof(msg), "%s: %s", what, why); return exl3_fail(ctx, code, msg); };
    if (!ctx) return EXL3_ERR_INVALID;
    if (a.bsz < 0 || a.q_len < 0 || a.rows < 0 || a.nq <= 0 || a.nkv <= 0 || a.pages <= 0 || a.pps <= 0 || a.pps > SPAN_MAX_LEN / EXL3_PAGE)
        return bad(EXL3_ERR_INVALID, "bad shape");
    if (!a.cu_q && (long long)a.bsz * a.q_len != a.rows) return bad(EXL3_ERR_INVALID, "rows must be bsz * q_len without cu_q");
    if (a.nq % a.nkv != 0) return bad(EXL3_ERR_INVALID, "n_q_heads must be a multiple of n_kv_heads");
    if ((long long)a.rows * a.nq > 1LL << 30) return bad(EXL3_ERR_INVALID, "too many rows");
    if (hd != 128) return bad(EXL3_ERR_UNSUPPORTED, "head_dim must be 128");
    if (!span_empty(a) && (!a.q || !a.o || !a.kc || !a.vc || !a.block_table || !a.seqlens)) return bad(EXL3_ERR_INVALID, "null argument");
    if (!aligned16(a.q) || !aligned16(a.o) || !aligned16(a.kc) || !aligned16(a.vc)) return bad(EXL3_ERR_INVALID, "pointers must be 16-byte aligned");
    if (!(sm_scale >= 0.f) || isinf(sm_scale)) return bad(EXL3_ERR_INVALID, "sm_scale must be finite and not negative");
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev != ctx->device) return bad(EXL3_ERR_INVALID, "the context's device must be the current one");
    return EXL3_OK;
}

int span_run(exl3_ctx* ctx, cudaStream_t st, const SpanArgs& a, const char* what)
{
    if (span_empty(a)) return EXL3_OK;
    const long long warps = (long long)a.rows * a.nq;
    exl3_launch_first(ctx, span_plain_kernel, (unsigned)((warps + 7) / 8), 256, 0, st, a);
    ctx->launches++;
    return exl3_check_launch(ctx, what);
}

}  // namespace

extern "C" int exl3_window_attn_paged(exl3_ctx* ctx, exl3_stream stream, const void* q, const void* k_cache, const void* v_cache,
                                      const int32_t* block_table, const int32_t* cache_seqlens, const int32_t* cu_q, void* o, int bsz,
                                      int q_len, int rows, int nq, int nkv, int hd, int pages, int pages_per_seq, int window, int sinks,
                                      float sm_scale)
{
    SpanArgs a = {(const half*)q, (half*)o, (const half*)k_cache, (const half*)v_cache, block_table, cache_seqlens, cu_q, nullptr, nullptr,
                  bsz, q_len, rows, nq, nkv, pages, pages_per_seq, 0, window, sinks, 0.f};
    const int rc = span_check(ctx, a, hd, sm_scale, "window_attn_paged");
    if (rc) return rc;
    EXL3_REQUIRE(window > 0 && sinks >= 0, "window_attn_paged: window must be positive and sinks not negative");
    a.scale_log2 = (sm_scale == 0.0f ? rsqrtf((float)hd) : sm_scale) * 1.4426950408889634f;
    return span_run(ctx, (cudaStream_t)stream, a, "window_attn_paged");
}

extern "C" int exl3_prefix_attn_paged(exl3_ctx* ctx, exl3_stream stream, const void* q, const void* k_cache, const void* v_cache,
                                      const int32_t* block_table, const int32_t* cache_seqlens, const int32_t* cu_q,
                                      const int32_t* group_start, const int32_t* prefix_lens, int n_groups, void* o, int bsz, int q_len,
                                      int rows, int nq, int nkv, int hd, int pages, int pages_per_seq, float sm_scale)
{
    SpanArgs a = {(const half*)q, (half*)o, (const half*)k_cache, (const half*)v_cache, block_table, cache_seqlens, cu_q, group_start, prefix_lens,
                  bsz, q_len, rows, nq, nkv, pages, pages_per_seq, n_groups, INT_MAX, 0, 0.f};
    const int rc = span_check(ctx, a, hd, sm_scale, "prefix_attn_paged");
    if (rc) return rc;
    EXL3_REQUIRE(n_groups >= 0 && n_groups <= bsz, "prefix_attn_paged: there are between 0 and bsz groups");
    EXL3_REQUIRE(n_groups == 0 || span_empty(a) || (group_start && prefix_lens), "prefix_attn_paged: null argument");
    a.scale_log2 = (sm_scale == 0.0f ? rsqrtf((float)hd) : sm_scale) * 1.4426950408889634f;
    return span_run(ctx, (cudaStream_t)stream, a, "prefix_attn_paged");
}
