// exl3_rope_append_paged / exl3_rope_append_paged_q: head norm and rotation of new queries and keys, the keys and values on their way
// into the pools, one launch.
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + bias)                       per head, where there is a norm weight
//   (u, v) -> (u cos a - v sin a, v cos a + u sin a) * attn_factor    for pair f < n_freq, a = inv_freq[f] * position of f's axis
//   q goes to out_q, k rotated and v as it is to their token's slot of the pools
//
// Everything between the fp16 input and the fp16 output is fp32, rounded once, but for the angle: at position 100 000 an fp32 product is
// off by 0.004 rad, so it is formed and reduced to half turns in 64 bits, once per row and frequency, and shared by all heads of the row
// through shared memory.
//
// What bounds it: HBM for many rows, the chain of dependent loads (row's sequence, length, page) and the launch for few.  A half warp
// holds a head, 8 values per lane and 16-byte accesses; a partner value of the half-split pairing comes by shuffle from the lane
// n_freq / 8 on.  The first values are requested ahead of the angles.
#include "common.cuh"
#include "kvquant.cuh"

namespace {

constexpr int RP_THREADS = 256, RP_HALF = RP_THREADS / 16;      // half warps: heads in work at a time
constexpr int RP_MAX_ROWS = 4;                                  // rows of a block: 64 frequencies each are the block's threads

struct RopePagedArgs {
    const half* q; half* out_q; const half* k; const half* v;
    const float* inv_freq;
    const int32_t* positions;                                   // [n_axes][rows], or NULL: the token's place in its sequence
    const half* q_norm; const half* k_norm;
    half* kc; half* vc;
    uint32_t* qk; half* sk; uint32_t* qv; half* sv;             // quantised pools
    const int32_t* block_table; const int32_t* seqlens; const int32_t* cu_q;
    float eps, cbias, attn_factor;
    int n_freq, mode, bsz, seq, rows, nq, nkv, pages, pps, k_bits, v_bits;
    uint8_t axis[64];
};

// R rows per block; heads of a row are taken by the block's half warps in turn, and by gridDim.y blocks.
template <int R, bool QUANT>
__global__ void __launch_bounds__(RP_THREADS) rope_paged_kernel(const RopePagedArgs a, int early)
{
    pdl_enter_first(early);
    __shared__ float2 s_cs[R][64];                              // cos, sin of a row's frequencies, times attn_factor
    __shared__ int s_pos[R];                                    // place in the sequence; -1: the row belongs to none
    __shared__ long long s_slot[R];                             // token slot in the pools; -1: none
    __shared__ __align__(16) half s_k[QUANT ? RP_HALF : 1][128];
    const int tid = threadIdx.x, lane = tid & 31, sub = tid & 15, hw = tid >> 4;
    const long long row0 = (long long)blockIdx.x * R;
    const int heads = a.nq + a.nkv, items = (int)min((long long)R, a.rows - row0) * heads;
    const int step = RP_HALF * gridDim.y;
    int item = (int)blockIdx.y * RP_HALF + hw;
    auto source = [&](int it) -> const half* {
        const long long row = row0 + it / heads;
        const int h = it % heads;
        return h < a.nq ? a.q + (row * a.nq + h) * 128 : a.k + (row * a.nkv + (h - a.nq)) * 128;
    };
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (item < items) raw = reinterpret_cast<const uint4*>(source(item))[sub];

    // every row's sequence, place and slot: a warp per row
    if (tid < R * 32 && row0 + (tid >> 5) < a.rows) {
        const int r = tid >> 5, row = (int)row0 + r;
        int b = -1, s = 0;
        if (a.cu_q) {                                           // cu_q[b] <= row < cu_q[b + 1]: the lanes probe the range side by side
            int lo = 0, hi = a.bsz;
            bool in = true;
            while (hi - lo > 1 && in) {
                const int width = (hi - lo + 31) >> 5, at = lo + lane * width;
                const unsigned below = __ballot_sync(0xffffffffu, at < hi && a.cu_q[at] <= row);
                in = below != 0;
                if (in) { lo += (31 - __clz(below)) * width; hi = min(hi, lo + width); }
            }
            if (in && a.cu_q[lo] <= row && row < a.cu_q[lo + 1] && a.cu_q[lo + 1] - a.cu_q[lo] <= a.seq) { b = lo; s = row - a.cu_q[lo]; }
        } else { b = row / a.seq; s = row - b * a.seq; }
        int pos = -1;
        long long slot = -1;
        if (b >= 0) {
            pos = a.seqlens[b] + s;
            if (pos >= 0 && (pos >> 8) < a.pps) {
                const int page = a.block_table[(size_t)b * a.pps + (pos >> 8)];
                if (page >= 0 && page < a.pages) slot = (long long)page * EXL3_PAGE + (pos & 255);
            }
            pos = max(pos, 0);
        }
        if (lane == 0) { s_pos[r] = pos; s_slot[r] = slot; }
    }
    __syncthreads();
    if (a.mode != EXL3_ROPE_NONE)
        for (int i = tid; i < R * 64; i += RP_THREADS) {
            const int r = i >> 6, f = i & 63;
            if (f < a.n_freq && row0 + r < a.rows) {
                const int pos = a.positions ? a.positions[(size_t)a.axis[f] * a.rows + row0 + r] : s_pos[r];
                double turn = (double)a.inv_freq[f] * (double)pos * 0.15915494309189533577;          // 1 / (2 pi)
                turn -= rint(turn);
                float sn, cs;
                sincospif(2.0f * (float)turn, &sn, &cs);
                s_cs[r][f] = make_float2(cs * a.attn_factor, sn * a.attn_factor);
            }
        }
    uint4 wq = make_uint4(0u, 0u, 0u, 0u), wk = wq;
    if (a.q_norm) wq = reinterpret_cast<const uint4*>(a.q_norm)[sub];
    if (a.k_norm) wk = reinterpret_cast<const uint4*>(a.k_norm)[sub];
    __syncthreads();

    // whole warps go round together (shuffles); a half warp behind the last item idles along
    for (int base = item - hw; base < items; base += step, item += step) {
        const bool on = item < items;
        const int it = on ? item : items - 1, r = it / heads, h = it % heads;
        const bool is_k = h >= a.nq;
        const uint4 x = raw;
        raw = make_uint4(0u, 0u, 0u, 0u);
        if (item + step < items) raw = reinterpret_cast<const uint4*>(source(item + step))[sub];
        float v[8];
        {
            const half2* p = reinterpret_cast<const half2*>(&x);
            #pragma unroll
            for (int j = 0; j < 4; ++j) { const float2 f = __half22float2(p[j]); v[2 * j] = f.x; v[2 * j + 1] = f.y; }
        }
        float ss = 0.f;
        #pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        #pragma unroll
        for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (is_k ? a.k_norm != nullptr : a.q_norm != nullptr) {
            const float inv = rsqrtf(ss * (1.0f / 128.0f) + a.eps);
            const uint4 w4 = is_k ? wk : wq;
            const half2* w = reinterpret_cast<const half2*>(&w4);
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __half22float2(w[j]);
                v[2 * j] *= inv * (f.x + a.cbias); v[2 * j + 1] *= inv * (f.y + a.cbias);
            }
        }
        if (a.mode == EXL3_ROPE_NEOX) {
            const int c = a.n_freq >> 3;                        // lanes of a half of the pairs
            const bool lower = sub < c, upper = !lower && sub < 2 * c;
            const int from = (lane & 16) | (lower ? sub + c : upper ? sub - c : sub);
            const float2* cs = s_cs[r] + 8 * (lower ? sub : upper ? sub - c : 0);
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float other = __shfl_sync(0xffffffffu, v[j], from);
                if (lower || upper) { const float2 t = cs[j]; v[j] = lower ? v[j] * t.x - other * t.y : v[j] * t.x + other * t.y; }
            }
        } else if (a.mode == EXL3_ROPE_GPTJ) {
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int f = 4 * sub + j;
                if (f < a.n_freq) {
                    const float2 t = s_cs[r][f];
                    const float u = v[2 * j], w = v[2 * j + 1];
                    v[2 * j] = u * t.x - w * t.y; v[2 * j + 1] = w * t.x + u * t.y;
                }
            }
        }
        uint4 y;
        {
            half2* p = reinterpret_cast<half2*>(&y);
            #pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        }
        const long long row = row0 + r, slot = s_slot[r];
        const bool live = on && s_pos[r] >= 0;
        if (live && !is_k) reinterpret_cast<uint4*>(a.out_q + (row * a.nq + h) * 128)[sub] = y;
        if constexpr (!QUANT) {
            if (live && is_k && slot >= 0) {
                const size_t at = ((size_t)slot * a.nkv + (h - a.nq)) * 16 + sub;
                reinterpret_cast<uint4*>(a.kc)[at] = y;
                reinterpret_cast<uint4*>(a.vc)[at] = reinterpret_cast<const uint4*>(a.v)[((size_t)row * a.nkv + (h - a.nq)) * 16 + sub];
            }
        } else {
            // the codec takes a whole warp per head: the warp's two heads one after the other, the key through shared memory
            const bool mine = live && is_k && slot >= 0;
            const unsigned any = __ballot_sync(0xffffffffu, mine);
            if (mine) reinterpret_cast<uint4*>(s_k[hw])[sub] = y;
            __syncwarp();
            #pragma unroll
            for (int side = 0; side < 2; ++side) {
                if (!(any >> (16 * side) & 1)) continue;                                 // warp-uniform
                const long long sl = __shfl_sync(0xffffffffu, slot, 16 * side);
                const int kv = __shfl_sync(0xffffffffu, h - a.nq, 16 * side);
                const long long rw = __shfl_sync(0xffffffffu, row, 16 * side);
                const size_t grp = ((size_t)sl * a.nkv + kv) * 4;
                exl3::quant_x4(s_k[(hw & ~1) + side], a.qk + grp * a.k_bits, a.sk + grp, 4, a.k_bits);
                exl3::quant_x4(a.v + ((size_t)rw * a.nkv + kv) * 128, a.qv + grp * a.v_bits, a.sv + grp, 4, a.v_bits);
            }
            __syncwarp();
        }
    }
}

int rope_append_impl(exl3_ctx* ctx, exl3_stream stream, RopePagedArgs& a, int n_axes, const uint8_t* freq_axis, int hd, bool quant)
{
    const bool empty = a.bsz == 0 || a.seq == 0 || a.rows == 0;            // touches none of its tensors
    EXL3_REQUIRE(ctx && (empty || (a.k && a.v && a.block_table && a.seqlens)), "rope_append_paged: null argument");
    EXL3_REQUIRE(a.bsz >= 0 && a.seq >= 0 && a.rows >= 0 && a.nq >= 0 && a.nkv > 0 && a.pages > 0 && a.pps > 0, "rope_append_paged: bad shape");
    EXL3_REQUIRE(a.q || a.nq == 0 || empty, "rope_append_paged: q is null but nq > 0");
    EXL3_REQUIRE(a.cu_q || (long long)a.bsz * a.seq == a.rows, "rope_append_paged: rows must be bsz * seq without cu_q");
    EXL3_REQUIRE((long long)a.rows * (a.nq + a.nkv) < (1LL << 40) && a.nq + a.nkv < (1 << 20), "rope_append_paged: too many heads");
    if (hd != 128) return exl3_fail(ctx, EXL3_ERR_UNSUPPORTED, "rope_append_paged: head_dim must be 128");
    EXL3_REQUIRE(a.mode == EXL3_ROPE_NEOX || a.mode == EXL3_ROPE_GPTJ || a.mode == EXL3_ROPE_NONE, "rope_append_paged: unknown rope_mode");
    if (a.mode != EXL3_ROPE_NONE) {
        EXL3_REQUIRE(a.inv_freq, "rope_append_paged: null inv_freq");
        EXL3_REQUIRE(a.n_freq > 0 && 2 * a.n_freq <= hd, "rope_append_paged: 2*n_freq must be <= head_dim");
        if (a.mode == EXL3_ROPE_NEOX && a.n_freq % 8 != 0)
            return exl3_fail(ctx, EXL3_ERR_UNSUPPORTED, "rope_append_paged: NEOX mode needs n_freq % 8 == 0");
        EXL3_REQUIRE(a.positions ? n_axes >= 1 && n_axes <= 255 : n_axes <= 1, "rope_append_paged: several axes need positions [n_axes, rows], one to 255 of them");
        memset(a.axis, 0, sizeof(a.axis));
        if (freq_axis)
            for (int f = 0; f < a.n_freq; ++f) {
                EXL3_REQUIRE(freq_axis[f] == 0 || freq_axis[f] < n_axes, "rope_append_paged: freq_axis names an axis that positions do not have");
                a.axis[f] = freq_axis[f];
            }
        else
            EXL3_REQUIRE(n_axes <= 1, "rope_append_paged: several axes need freq_axis");
    }
    EXL3_REQUIRE(aligned16(a.q) && aligned16(a.out_q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.q_norm) && aligned16(a.k_norm),
                 "rope_append_paged: pointers must be 16-byte aligned");
    int dev = -1;
    EXL3_REQUIRE(cudaGetDevice(&dev) == cudaSuccess && dev == ctx->device, "rope_append_paged: the context's device must be the current one");
    if (empty) return EXL3_OK;
    if (!a.out_q) a.out_q = const_cast<half*>(a.q);
    const int heads = a.nq + a.nkv;
    // Four rows per block share the work on angles evenly; where that leaves SMs idle, a row per block, its heads over several blocks
    const bool many = a.rows >= RP_MAX_ROWS * 4 * ctx->num_sms;
    const dim3 grid(many ? (a.rows + RP_MAX_ROWS - 1) / RP_MAX_ROWS : a.rows,
                    many ? 1 : (unsigned)max(1, min((heads + RP_HALF - 1) / RP_HALF, 4 * ctx->num_sms / a.rows)));
    cudaStream_t st = (cudaStream_t)stream;
    if (quant) {
        if (many) exl3_launch_first(ctx, rope_paged_kernel<RP_MAX_ROWS, true>, grid, RP_THREADS, 0, st, a);
        else exl3_launch_first(ctx, rope_paged_kernel<1, true>, grid, RP_THREADS, 0, st, a);
    } else {
        if (many) exl3_launch_first(ctx, rope_paged_kernel<RP_MAX_ROWS, false>, grid, RP_THREADS, 0, st, a);
        else exl3_launch_first(ctx, rope_paged_kernel<1, false>, grid, RP_THREADS, 0, st, a);
    }
    ctx->launches++;
    return exl3_check_launch(ctx, "rope_append_paged");
}

}  // namespace

extern "C" int exl3_rope_append_paged(exl3_ctx* ctx, exl3_stream stream, const void* q, void* out_q, const void* k, const void* v,
                                      const float* inv_freq, int n_freq, const int32_t* positions, int n_axes, const uint8_t* freq_axis,
                                      const void* q_norm, const void* k_norm, float norm_eps, float norm_constant_bias, int rope_mode,
                                      float attn_factor, void* k_cache, void* v_cache, const int32_t* block_table,
                                      const int32_t* cache_seqlens, const int32_t* cu_q, int bsz, int seq, int rows, int nq, int nkv, int hd,
                                      int pages, int pages_per_seq)
{
    EXL3_REQUIRE(ctx && k_cache && v_cache, "rope_append_paged: null argument");
    EXL3_REQUIRE(aligned16(k_cache) && aligned16(v_cache), "rope_append_paged: pointers must be 16-byte aligned");
    RopePagedArgs a = {(const half*)q, (half*)out_q, (const half*)k, (const half*)v, inv_freq, positions, (const half*)q_norm, (const half*)k_norm,
                       (half*)k_cache, (half*)v_cache, nullptr, nullptr, nullptr, nullptr, block_table, cache_seqlens, cu_q,
                       norm_eps, norm_constant_bias, attn_factor, n_freq, rope_mode, bsz, seq, rows, nq, nkv, pages, pages_per_seq, 0, 0, {}};
    return rope_append_impl(ctx, stream, a, n_axes, freq_axis, hd, false);
}

extern "C" int exl3_rope_append_paged_q(exl3_ctx* ctx, exl3_stream stream, const void* q, void* out_q, const void* k, const void* v,
                                        const float* inv_freq, int n_freq, const int32_t* positions, int n_axes, const uint8_t* freq_axis,
                                        const void* q_norm, const void* k_norm, float norm_eps, float norm_constant_bias, int rope_mode,
                                        float attn_factor, void* qk, void* sk, void* qv, void* sv, const int32_t* block_table,
                                        const int32_t* cache_seqlens, const int32_t* cu_q, int bsz, int seq, int rows, int nq, int nkv, int hd,
                                        int pages, int pages_per_seq, int k_bits, int v_bits)
{
    EXL3_REQUIRE(ctx && qk && sk && qv && sv, "rope_append_paged: null argument");
    EXL3_REQUIRE(k_bits >= 2 && k_bits <= 8 && v_bits >= 2 && v_bits <= 8, "rope_append_paged: bits must be 2..8");
    EXL3_REQUIRE(quant_planes_aligned(qk, sk, qv, sv), "rope_append_paged: code planes must be 16-byte and scale planes 8-byte aligned");
    RopePagedArgs a = {(const half*)q, (half*)out_q, (const half*)k, (const half*)v, inv_freq, positions, (const half*)q_norm, (const half*)k_norm,
                       nullptr, nullptr, (uint32_t*)qk, (half*)sk, (uint32_t*)qv, (half*)sv, block_table, cache_seqlens, cu_q,
                       norm_eps, norm_constant_bias, attn_factor, n_freq, rope_mode, bsz, seq, rows, nq, nkv, pages, pages_per_seq, k_bits, v_bits, {}};
    return rope_append_impl(ctx, stream, a, n_axes, freq_axis, hd, true);
}
