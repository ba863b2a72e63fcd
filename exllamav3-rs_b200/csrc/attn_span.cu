// exl3_window_attn_paged and exl3_prefix_attn_paged: attention over spans of the paged cache.
#include <limits.h>
#include <math.h>
#include "attn_span.cuh"
#include "attn_rows.cuh"

namespace {

using namespace exl3;

// The plain kernel: a warp per (row, head), one key at a time, lane = 4 dims.  Sequences with more than `few` (query, head) rows per kv head.
__global__ void __launch_bounds__(256) span_plain_kernel(const SpanArgs a, int few, int early)
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
    if (row < s.row_base || row >= s.row_base + s.ql || s.ql * (a.nq / a.nkv) <= few) return;
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

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn span_encode_tiled()
{
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)ptr;
        else
            cudaGetLastError();
    }
    return fn;
}

// A pool as {64 dims, 256 tokens, 2 halves of a head, heads, pages}: a box of `tokens` and `halves` lands as halves of 128-byte rows in the
// 128-byte swizzle.
bool span_map(const SpanArgs& a, const void* pool, int tokens, int halves, CUtensorMap* map)
{
    EncodeTiledFn enc = span_encode_tiled();
    if (!enc) return false;
    const cuuint64_t tok = (cuuint64_t)a.nkv * 256;
    cuuint64_t dims[5] = {64, EXL3_PAGE, 2, (cuuint64_t)a.nkv, (cuuint64_t)a.pages};
    cuuint64_t strides[4] = {tok, 128, 256, EXL3_PAGE * tok};
    cuuint32_t box[5] = {64, (cuuint32_t)tokens, (cuuint32_t)halves, 1, 1};
    cuuint32_t one[5] = {1, 1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(pool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename Kern>
bool span_configure(Kern kern, int bytes, int device, bool (&done)[64])
{
    if (device >= 0 && device < 64 && done[device]) return true;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) { cudaGetLastError(); return false; }
    if (device >= 0 && device < 64) done[device] = true;
    return true;
}

// the sequences of few rows
int span_rows(exl3_ctx* ctx, cudaStream_t st, const SpanArgs& a, bool first, size_t* ws_off)
{
    ArMaps maps;
    if (!span_map(a, a.kc, AR_TK, 2, &maps.k) || !span_map(a, a.vc, AR_TK, 2, &maps.v) || !span_map(a, a.kc, 16, 1, &maps.k16) || !span_map(a, a.vc, 16, 1, &maps.v16))
        return exl3_fail(ctx, EXL3_ERR_CUDA, "attention: no tensor map of the pools");
    static bool done[64] = {};
    if (!span_configure(attn_rows_kernel, ArSmem::BYTES, ctx->device, done)) return exl3_fail(ctx, EXL3_ERR_CUDA, "attention: shared memory");
    const int ctas = 2 * ctx->num_sms;
    ArParams p;
    p.a = a; p.min_share = 2;
    p.partial = (float*)exl3_ws_take(ctx, ws_off, (size_t)2 * ctas * AR_ROWS * AR_MS * 4);
    if (!p.partial) return exl3_fail(ctx, EXL3_ERR_WORKSPACE, "attention: context scratch too small for the partial sums");
    p.counters = ctx->counters; p.status = ctx->status;
    for (int b0 = 0; b0 < a.bsz; b0 += AR_MAX_BSZ) {
        p.b0 = b0; p.bsz = min(AR_MAX_BSZ, a.bsz - b0);
        p.first = first || b0 > 0;                          // launches of one call share the partial sums
        // no more CTAs than there can be shares: a sequence has at most the tiles of its window and first keys, or of its table
        const long long most = min((long long)a.pps * (EXL3_PAGE / AR_TK),
                                   ((long long)min(a.window, SPAN_MAX_LEN) + AR_ROWS) / AR_TK + 2 + min(a.sinks, SPAN_MAX_LEN) / AR_TK + 1);
        const int grid = (int)min((long long)ctas, max(1LL, (most * p.bsz * a.nkv + p.min_share - 1) / p.min_share));
        if (p.first) exl3_launch_first(ctx, attn_rows_kernel, grid, AR_THREADS, ArSmem::BYTES, st, maps, p);
        else exl3_launch(ctx, attn_rows_kernel, grid, AR_THREADS, ArSmem::BYTES, st, maps, p, 0);
        ctx->launches++;
    }
    return EXL3_OK;
}

int span_run(exl3_ctx* ctx, cudaStream_t st, const SpanArgs& a, const char* what)
{
    if (span_empty(a)) return EXL3_OK;
    size_t off = 0;
    const int G = a.nq / a.nkv;
    const bool few = G <= AR_ROWS && a.n_groups == 0;
    if (few) {
        const int rc = span_rows(ctx, st, a, true, &off);
        if (rc) return rc;
    }
    if (!few || (long long)a.q_len * G > AR_ROWS) {
        const long long warps = (long long)a.rows * a.nq;
        exl3_launch_first(ctx, span_plain_kernel, (unsigned)((warps + 7) / 8), 256, 0, st, a, few ? AR_ROWS : 0);
        ctx->launches++;
    }
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
