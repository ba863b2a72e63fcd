// exl3_window_attn_paged and exl3_prefix_attn_paged: attention over spans of the paged cache.
#include <algorithm>
#include <cmath>
#include <limits.h>
#include <math.h>
#include "attn_span_tc.cuh"

namespace {

using namespace exl3;

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
    if (a.nq / a.nkv > AS_BLOCK) return bad(EXL3_ERR_UNSUPPORTED, "more than 128 query heads per kv head");
    if (a.bsz > 32 * AS_MAX_CHUNKS) return bad(EXL3_ERR_UNSUPPORTED, "more than 8192 sequences");
    if ((long long)a.rows * a.nq > 1LL << 30) return bad(EXL3_ERR_INVALID, "too many rows");
    if (hd != 128) return bad(EXL3_ERR_UNSUPPORTED, "head_dim must be 128");
    // The kernels count key tiles in 32 bits: of 16 keys over the sequences of a launch, of 128 keys over a head's row blocks (a block has more
    // than half of its rows)
    const double keys = std::min((double)a.pps * EXL3_PAGE, (double)a.window + a.sinks + a.q_len) + 512;
    const double blocks = (double)a.rows * (a.nq / a.nkv) / (AS_BLOCK / 2) + a.bsz;
    if (std::min(a.bsz, AR_MAX_BSZ) * keys / 16 >= 2147483648.0 || blocks * keys / AS_TK >= 2147483648.0)
        return bad(EXL3_ERR_UNSUPPORTED, "rows and block tables of more than 2^31 key tiles");
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

// A pool as {64 dims, 256 tokens, 2 halves of a head, heads, pages}: a box lands as heads of halves of 128-byte rows, a row per token, in
// the 128-byte swizzle.
bool span_map(const SpanArgs& a, const void* pool, int tokens, int halves, int heads, CUtensorMap* map)
{
    EncodeTiledFn enc = span_encode_tiled();
    if (!enc) return false;
    const cuuint64_t tok = (cuuint64_t)a.nkv * 256;
    cuuint64_t dims[5] = {64, EXL3_PAGE, 2, (cuuint64_t)a.nkv, (cuuint64_t)a.pages};
    cuuint64_t strides[4] = {tok, 128, 256, EXL3_PAGE * tok};
    cuuint32_t box[5] = {64, (cuuint32_t)tokens, (cuuint32_t)halves, (cuuint32_t)heads, 1};
    cuuint32_t one[5] = {1, 1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(pool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The queries as {64 dims, 2 halves, heads, rows}: a box of a kv head's G heads and so many rows lands as packed rows
bool span_q_map(const SpanArgs& a, int rows, CUtensorMap* map)
{
    EncodeTiledFn enc = span_encode_tiled();
    if (!enc) return false;
    const int G = a.nq / a.nkv;
    cuuint64_t dims[4] = {64, 2, (cuuint64_t)a.nq, (cuuint64_t)a.rows};
    cuuint64_t strides[3] = {128, 256, (cuuint64_t)a.nq * 256};
    cuuint32_t box[4] = {64, 1, (cuuint32_t)G, (cuuint32_t)(rows / G)};
    cuuint32_t one[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<half*>(a.q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
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

// the sequences of few rows, HW heads side by side
constexpr size_t AR_SCRATCH = (size_t)AR_WARPS * AR_ROWS * AR_MS * 4;       // per CTA and place, at most
// Keys that a CTA takes at least: fewer are more partial sums to join (us at 64, 128 and 192 keys: one row over a window of 1024 16.2, 15.5 and
// 20.7, of 4096 26, 20 and 23)
constexpr int AR_MIN_KEYS = 128;
template <int HW, bool ALONE, bool BESIDE = false>
int span_rows(exl3_ctx* ctx, cudaStream_t st, const SpanArgs& a, bool first, bool plain, const AsParams& pre, int sms, size_t* ws_off)
{
    using Cfg = ArCfg<HW>;
    ArMaps maps;
    if (!span_map(a, a.kc, Cfg::TK, 2, HW, &maps.k) || !span_map(a, a.vc, Cfg::TK, 2, HW, &maps.v) ||
        (Cfg::KW > 1 && (!span_map(a, a.kc, 16, 1, 1, &maps.k16) || !span_map(a, a.vc, 16, 1, 1, &maps.v16))))
        return exl3_fail(ctx, EXL3_ERR_CUDA, "attention: no tensor map of the pools");
    if (Cfg::KW == 1) { maps.k16 = maps.k; maps.v16 = maps.v; }
    static bool done[64] = {};
    if (!span_configure(attn_rows_kernel<HW, ALONE, BESIDE>, Cfg::BYTES, ctx->device, done)) return exl3_fail(ctx, EXL3_ERR_CUDA, "attention: shared memory");
    const int ctas = sms;
    ArParams p;
    p.a = a;
    p.min_share = AR_MIN_KEYS / Cfg::TK;
    p.partial = (float*)exl3_ws_take(ctx, ws_off, 2 * ctas * AR_SCRATCH);
    if (!p.partial) return exl3_fail(ctx, EXL3_ERR_WORKSPACE, "attention: context scratch too small for the partial sums");
    p.counters = ctx->counters; p.status = ctx->status;
    p.rest = pre.rest;
    for (int b0 = 0; b0 < a.bsz; b0 += AR_MAX_BSZ) {
        p.b0 = b0; p.bsz = std::min(AR_MAX_BSZ, a.bsz - b0);
        p.first = first || b0 > 0;                          // launches of one call share the partial sums
        // no more CTAs than there can be shares: a sequence has at most the tiles of its window and first keys, or of its table
        const long long most = std::min((long long)a.pps * (EXL3_PAGE / Cfg::TK),
                                        ((long long)std::min(a.window, SPAN_MAX_LEN) + AR_ROWS) / Cfg::TK + 2 + std::min(a.sinks, SPAN_MAX_LEN) / Cfg::TK + 1) + 1;
        const int grid = BESIDE ? ctas : (int)std::min((long long)ctas, std::max(1LL, (most * p.bsz * (a.nkv / HW) + p.min_share - 1) / p.min_share));
        if (p.first && !plain) exl3_launch_first(ctx, attn_rows_kernel<HW, ALONE, BESIDE>, grid, AR_THREADS, Cfg::BYTES, st, maps, p);
        else exl3_launch(ctx, attn_rows_kernel<HW, ALONE, BESIDE>, grid, AR_THREADS, Cfg::BYTES, st, maps, p, 0);
        ctx->launches++;
    }
    return EXL3_OK;
}

// a launch of the tcgen05 kernel with NB row blocks per CTA
template <int NB, bool BESIDE = false>
int span_tc(exl3_ctx* ctx, cudaStream_t st, const AsParams& p, int sms)
{
    CUtensorMap kmap, vmap, qmap;
    if (!span_map(p.a, p.a.kc, AS_TK, 2, 1, &kmap) || !span_map(p.a, p.a.vc, AS_TK, 2, 1, &vmap) || !span_q_map(p.a, AsCfg<NB>::ROWS, &qmap))
        return exl3_fail(ctx, EXL3_ERR_CUDA, "attention: no tensor map of the pools");
    static bool done[64] = {};
    if (!span_configure(attn_span_kernel<NB, BESIDE>, AsCfg<NB>::SMEM, ctx->device, done)) return exl3_fail(ctx, EXL3_ERR_CUDA, "attention: shared memory");
    const int grid = AsCfg<NB>::CTAS * sms;
    if (p.first) exl3_launch_first(ctx, attn_span_kernel<NB, BESIDE>, grid, AsCfg<NB>::THREADS, AsCfg<NB>::SMEM, st, kmap, vmap, qmap, p);
    else exl3_launch(ctx, attn_span_kernel<NB, BESIDE>, grid, AsCfg<NB>::THREADS, AsCfg<NB>::SMEM, st, kmap, vmap, qmap, p, 0);
    ctx->launches++;
    return EXL3_OK;
}

// Whether a batch over windows may have both classes, and enough of them that their kernels run beside one another, each on the SMs that
// span_few_sms gives it: as far as the host knows, by full windows.
bool span_beside(exl3_ctx* ctx, const SpanArgs& a)
{
    if (a.n_groups > 0 || a.window > SPAN_MAX_LEN || a.q_len < 2 || a.bsz > AR_MAX_BSZ) return false;
    const int G = a.nq / a.nkv;
    const double tiles = std::min((double)a.window + a.sinks, (double)a.pps * EXL3_PAGE) / AS_TK;
    const double n_long = std::max(0.0, std::ceil(((double)a.rows - a.bsz) / (a.q_len - 1))), n_few = a.bsz - n_long;
    const double few = n_few * tiles * a.nkv * SPAN_FEW_TILE / 20;                                         // us of one SM
    const double many = n_long * std::ceil((double)a.q_len * G / 256) * a.nkv * (tiles * SPAN_MANY_TILE + SPAN_MANY_UNIT) / 20;
    return n_long >= 1 && n_few >= 1 && few >= many / 16 && many >= few / 16 && few + many >= 10.0 * ctx->num_sms;
}

int span_run(exl3_ctx* ctx, cudaStream_t st, const SpanArgs& a, const char* what)
{
    if (span_empty(a)) return EXL3_OK;
    const int G = a.nq / a.nkv;
    const long long packed = (long long)a.q_len * G, all = (long long)a.rows * G;
    const bool any_long = packed > AR_ROWS, any_few = G <= AR_ROWS && (a.cu_q || !any_long);
    // A few sequences of few rows read a short prefix sooner each than together, which is two kernels more: up to 128 MB read again, as far as the
    // host knows, which is the table's width: tables much wider than the prefix take the way together.  us, each and together, 16 / 8 heads,
    // sequences x prefix: 4 x 512 17 and 27, 8 x 2048 24 and 31, 16 x 2048 35 and 38, 32 x 1024 37 and 29; 40 / 8 heads: 4 x 8192 42 and 39,
    // 8 x 8192 57 and 41.
    const bool alone = a.n_groups > 0 && !any_long && (double)(a.bsz - 1) * a.pps * EXL3_PAGE * a.nkv * 512 <= 128.0 * (1 << 20);
    const bool groups = a.n_groups > 0 && !alone;
    // Two row blocks share the tiles where a group or a sequence may have that many rows
    const bool two_prefix = all > (long long)AS_BLOCK * a.n_groups, two_own = packed > AS_BLOCK;
    // Scratch.  Prefixes: a place per row, head and part, as many parts as a quarter of the scratch has room for, and one for
    // the sequence's rest.  Own spans: two units per CTA.
    const size_t place = (size_t)a.rows * a.nq * SPAN_PART * 4;
    AsParams p = {a, 0, nullptr, nullptr, (int)std::max((size_t)1, std::min((size_t)AS_MAX_SPLITS, ctx->ws_bytes / 4 / place)), nullptr,
                  ctx->counters + 4096, ctx->status, 1};
    size_t off = 0;
    int* share = (int*)exl3_ws_take(ctx, &off, 2 * sizeof(int));
    float* prefix = groups ? (float*)exl3_ws_take(ctx, &off, place * p.max_splits) : nullptr;
    if (groups) p.rest = (float*)exl3_ws_take(ctx, &off, place);
    float* own = any_long ? (float*)exl3_ws_take(ctx, &off, (size_t)2 * ctx->num_sms * 2 * AS_BLOCK * SPAN_PART * 4) : nullptr;
    size_t probe = off;
    if (!share || (groups && (!prefix || !p.rest)) || (any_long && !own) || (any_few && !exl3_ws_take(ctx, &probe, (size_t)2 * ctx->num_sms * AR_SCRATCH)))
        return exl3_fail(ctx, EXL3_ERR_WORKSPACE, "attention: context scratch too small for the partial sums");
    int rc = EXL3_OK;
    if (groups) {
        p.prefixes = 1; p.partial = prefix; p.share = share;
        rc = two_prefix ? span_tc<2>(ctx, st, p, ctx->num_sms) : span_tc<1>(ctx, st, p, ctx->num_sms);
        if (rc) return rc;
        p.first = 0;
    }
    exl3_chain_scope chain(ctx, groups);
    // Both classes of a batch over windows: each gets its share of the SMs, and the start and end of one kernel, 10 us and more, runs under the
    // other (us, and one call of each class behind the other: 28 rows beside 4 x 251, window 1024 92 and 93, 64 x 1 beside 2 x 300, window 2048 91 and 103, 28 x 1
    // beside 251, window 4096 125 and 142; 40 x 1 at 200 tokens beside 512 at 16384 91 and 91, 120 x 1 at 20 to 300 beside 4 x 1024, window 4096 461 and 426).
    const bool beside = any_long && any_few && span_beside(ctx, a);
    SpanArgs both = a;
    if (beside) {
        both.beside = ctx->num_sms; both.unit_rows = AS_BLOCK * (two_own ? 2 : 1) / G * G;
        p.a = both;
        if (cudaEventRecord(ctx->ev_fork, st) != cudaSuccess || cudaStreamWaitEvent(ctx->aux_stream, ctx->ev_fork, 0) != cudaSuccess)
            return exl3_fail(ctx, EXL3_ERR_CUDA, "attention: stream fork failed");
        const int chained = ctx->chain;
        ctx->chain = 0;                                      // a plain launch: nothing of the second stream is in front
        rc = a.nkv % 4 == 0 ? span_rows<4, false, true>(ctx, ctx->aux_stream, both, true, true, p, ctx->num_sms, &off)
                            : span_rows<1, false, true>(ctx, ctx->aux_stream, both, true, true, p, ctx->num_sms, &off);
        ctx->chain = chained;
        ctx->chain_break = 1;
    }
    if (any_long && rc == EXL3_OK) {
        p.prefixes = 0; p.partial = own; p.share = share + 1;
        rc = beside ? two_own ? span_tc<2, true>(ctx, st, p, ctx->num_sms) : span_tc<1, true>(ctx, st, p, ctx->num_sms)
                    : two_own ? span_tc<2>(ctx, st, p, ctx->num_sms) : span_tc<1>(ctx, st, p, ctx->num_sms);
        p.first = 0;
    }
    if (beside) {
        // joined after an error too, so that a capture in progress stays well-formed
        if (cudaEventRecord(ctx->ev_join, ctx->aux_stream) != cudaSuccess || cudaStreamWaitEvent(st, ctx->ev_join, 0) != cudaSuccess)
            return exl3_fail(ctx, EXL3_ERR_CUDA, "attention: stream join failed");
        return rc ? rc : exl3_check_launch(ctx, what);
    }
    if (rc) return rc;
    exl3_chain_scope behind(ctx, any_long);
    if (any_few) {
        const bool four = a.nkv % 4 == 0, first = p.first != 0;
        rc = alone ? four ? span_rows<4, true>(ctx, st, a, first, false, p, ctx->num_sms, &off) : span_rows<1, true>(ctx, st, a, first, false, p, ctx->num_sms, &off)
                   : four ? span_rows<4, false>(ctx, st, a, first, false, p, ctx->num_sms, &off) : span_rows<1, false>(ctx, st, a, first, false, p, ctx->num_sms, &off);
        if (rc) return rc;
    }
    if (groups) {
        const SpanJoinParams j = {a, prefix, share, p.rest};
        const long long pairs = (long long)a.rows * a.nq;
        // us, whole calls, one pair per warp and four: 64 x 16 pairs 69 and 74, 1024 x 40 pairs 884 and 846
        if (pairs <= 64LL * ctx->num_sms) exl3_launch(ctx, span_join_kernel<1>, (unsigned)((pairs + 7) / 8), 256, 0, st, j);
        else exl3_launch(ctx, span_join_kernel<4>, (unsigned)((pairs + 31) / 32), 256, 0, st, j);
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
                  bsz, q_len, rows, nq, nkv, pages, pages_per_seq, 0, window, sinks, 0.f, 0, 0};
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
                  bsz, q_len, rows, nq, nkv, pages, pages_per_seq, n_groups, INT_MAX, 0, 0.f, 0, 0};
    const int rc = span_check(ctx, a, hd, sm_scale, "prefix_attn_paged");
    if (rc) return rc;
    EXL3_REQUIRE(n_groups >= 0 && n_groups <= bsz, "prefix_attn_paged: there are between 0 and bsz groups");
    EXL3_REQUIRE(n_groups == 0 || span_empty(a) || (group_start && prefix_lens), "prefix_attn_paged: null argument");
    a.scale_log2 = (sm_scale == 0.0f ? rsqrtf((float)hd) : sm_scale) * 1.4426950408889634f;
    return span_run(ctx, (cudaStream_t)stream, a, "prefix_attn_paged");
}
