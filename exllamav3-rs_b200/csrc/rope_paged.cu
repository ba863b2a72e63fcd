// exl3_rope_append_paged: head norm and rotation of new queries and keys, the keys and values on their way
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
// What bounds it: for few rows the launch and the chain of dependent loads (row's sequence, length, page): 1 and 64 rows 5.1 and 5.3 us, cold caches,
// under 9 and 9.6 us of a call's host side.  8192 rows of 40 / 8 heads: 48 to 52 us, 4.5 to 4.8 TB/s; issue slots 61 % and DRAM 46 % busy, and 1024 blocks
// on 592 places, so neither alone (`profiles/`).  8192 rows into 4- and 8-bit pools 90 and 86 us, 40 and 37 of them the codec's.  A half warp
// holds a head, 8 values per lane and 16-byte accesses; a partner value of the half-split pairing comes by shuffle from the lane
// n_freq / 8 on.  Values are requested a head ahead, of two rows at a time where there are many, the first ones ahead of the angles.
#include "common.cuh"
#include "kvquant.cuh"

namespace {

constexpr int RP_THREADS = 256, RP_HALF = RP_THREADS / 16;      // half warps: heads in work at a time
constexpr int RP_ROWS = 8;                                      // rows of a block where there are many

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

// R rows per block, B of them in work together; a row's heads are taken by the block's half warps, and by gridDim.y blocks.
template <int R, int B, bool QUANT>
__global__ void __launch_bounds__(RP_THREADS, 4) rope_paged_kernel(const RopePagedArgs a, int early)
{
    pdl_enter_first(early);
    // cos, sin of a row's frequencies, times attn_factor, as the lanes read them: pairs of frequencies, the pairs of all lanes side by side
    // (frequency after frequency, a lane's 64 bytes apart, the reads' bank conflicts were what 8192 rows waited for: 68 us, and 51 without)
    __shared__ __align__(16) float4 s_cs[R][32];
    __shared__ int s_pos[R];                                    // place in the sequence; -1: the row belongs to none
    __shared__ long long s_slot[R];                             // token slot in the pools; -1: none
    __shared__ __align__(16) half s_k[QUANT ? RP_HALF : 1][128];
    const int tid = threadIdx.x, lane = tid & 31, sub = tid & 15, hw = tid >> 4;
    const long long row0 = (long long)blockIdx.x * R;
    const int heads = a.nq + a.nkv, step = RP_HALF * gridDim.y;
    int h = (int)blockIdx.y * RP_HALF + hw;
    const int there = (int)min((long long)R, a.rows - row0);    // rows of this block
    auto load = [&](uint4 (&x)[B], int r0, int h) {
        const half* src = h < a.nq ? a.q + ((row0 + r0) * a.nq + h) * 128 : a.k + ((row0 + r0) * a.nkv + (h - a.nq)) * 128;
        const size_t next = (size_t)(h < a.nq ? a.nq : a.nkv) * 16;
        #pragma unroll
        for (int i = 0; i < B; ++i) {
            x[i] = make_uint4(0u, 0u, 0u, 0u);
            if (h < heads && r0 + i < there) x[i] = reinterpret_cast<const uint4*>(src)[i * next + sub];
        }
    };
    uint4 ahead[B];
    load(ahead, 0, h);

    // every row's sequence, place and slot: a warp per row
    if ((tid >> 5) < there) {
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
            if (in) {
                const int from = a.cu_q[lo], to = a.cu_q[lo + 1];
                if (from <= row && row < to && to - from <= a.seq) { b = lo; s = row - from; }
            }
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
    uint4 wq = make_uint4(0u, 0u, 0u, 0u), wk = wq;
    if (a.q_norm) wq = reinterpret_cast<const uint4*>(a.q_norm)[sub];
    if (a.k_norm) wk = reinterpret_cast<const uint4*>(a.k_norm)[sub];
    // angles: positions of their own need no sequence
    if (!a.positions) __syncthreads();
    if (a.mode != EXL3_ROPE_NONE)
        for (int i = tid; i < R * 64; i += RP_THREADS) {
            const int r = i >> 6, f = i & 63;
            if (f < a.n_freq && r < there) {
                const int pos = a.positions ? a.positions[(size_t)a.axis[f] * a.rows + row0 + r] : s_pos[r];
                double turn = (double)a.inv_freq[f] * (double)pos * 0.15915494309189533577;          // 1 / (2 pi)
                turn -= rint(turn);
                float sn, cs;
                sincospif(2.0f * (float)turn, &sn, &cs);
                const int pair = a.mode == EXL3_ROPE_NEOX ? ((f & 7) >> 1) * 8 + (f >> 3) : ((f & 3) >> 1) * 16 + (f >> 2);
                reinterpret_cast<float2*>(&s_cs[r][pair])[f & 1] = make_float2(cs * a.attn_factor, sn * a.attn_factor);
            }
        }
    __syncthreads();

    // whole warps go round together (shuffles); a half warp behind the last head idles along
    const int h0 = h, c = a.n_freq >> 3;                        // NEOX: lanes of a half of the pairs
    const bool lower = sub < c, upper = !lower && sub < 2 * c;
    const int from = (lane & 16) | (lower ? sub + c : upper ? sub - c : sub);
    for (int r0 = 0; r0 < there;) {
        const bool on = h < heads, is_k = h >= a.nq;
        uint4 x[B], vv[B];
        #pragma unroll
        for (int i = 0; i < B; ++i) { x[i] = ahead[i]; vv[i] = make_uint4(0u, 0u, 0u, 0u); }
        const int h_now = h, r_now = r0;
        h += step;
        if (h - hw >= heads) { h = h0; r0 += B; }               // the next rows' first head (whole blocks agree)
        load(ahead, r0, h);
        if (!QUANT && on && is_k) {
            #pragma unroll
            for (int i = 0; i < B; ++i)
                if (r_now + i < there) vv[i] = reinterpret_cast<const uint4*>(a.v)[((row0 + r_now + i) * a.nkv + (h_now - a.nq)) * 16 + sub];
        }
        const bool norm = is_k ? a.k_norm != nullptr : a.q_norm != nullptr;
        #pragma unroll
        for (int i = 0; i < B; ++i) {
            const int r = min(r_now + i, R - 1);
            float v[8];
            {
                const half2* p = reinterpret_cast<const half2*>(&x[i]);
                #pragma unroll
                for (int j = 0; j < 4; ++j) { const float2 f = __half22float2(p[j]); v[2 * j] = f.x; v[2 * j + 1] = f.y; }
            }
            if (a.q_norm || a.k_norm) {                         // the same for the whole grid
                float ss = 0.f;
                #pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
                #pragma unroll
                for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (norm) {
                    const float inv = rsqrtf(ss * (1.0f / 128.0f) + a.eps);
                    const uint4 w4 = is_k ? wk : wq;
                    const half2* w = reinterpret_cast<const half2*>(&w4);
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 f = __half22float2(w[j]);
                        v[2 * j] *= inv * (f.x + a.cbias); v[2 * j + 1] *= inv * (f.y + a.cbias);
                    }
                }
            }
            if (a.mode == EXL3_ROPE_NEOX) {
                const float4* cs = s_cs[r] + (lower ? sub : upper ? sub - c : 0);
                #pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float o0 = __shfl_sync(0xffffffffu, v[j], from), o1 = __shfl_sync(0xffffffffu, v[j + 1], from);
                    if (lower || upper) {
                        const float4 t = cs[(j >> 1) * 8];
                        v[j] = fmaf(v[j], t.x, lower ? -o0 * t.y : o0 * t.y);
                        v[j + 1] = fmaf(v[j + 1], t.z, lower ? -o1 * t.w : o1 * t.w);
                    }
                }
            } else if (a.mode == EXL3_ROPE_GPTJ) {
                #pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    const float4 t = s_cs[r][(j >> 1) * 16 + sub];
                    #pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (4 * sub + j + k < a.n_freq) {
                            const float u = v[2 * (j + k)], w = v[2 * (j + k) + 1], cs = k ? t.z : t.x, sn = k ? t.w : t.y;
                            v[2 * (j + k)] = u * cs - w * sn; v[2 * (j + k) + 1] = w * cs + u * sn;
                        }
                }
            }
            uint4 y;
            {
                half2* p = reinterpret_cast<half2*>(&y);
                #pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            }
            const bool live = on && r_now + i < there && s_pos[r] >= 0;
            const long long row = row0 + r, slot = live ? s_slot[r] : -1;
            if (live && !is_k) reinterpret_cast<uint4*>(a.out_q + (row * a.nq + h_now) * 128)[sub] = y;
            if constexpr (!QUANT) {
                if (live && is_k && slot >= 0) {
                    const size_t at = ((size_t)slot * a.nkv + (h_now - a.nq)) * 16 + sub;
                    reinterpret_cast<uint4*>(a.kc)[at] = y;
                    reinterpret_cast<uint4*>(a.vc)[at] = vv[i];
                }
            } else {
                // the codec takes a whole warp per head: the warp's two heads one after the other, the key through shared memory
                const bool mine = live && is_k && slot >= 0;
                const unsigned any = __ballot_sync(0xffffffffu, mine);
                if (mine) reinterpret_cast<uint4*>(s_k[hw])[sub] = y;
                __syncwarp();
                #pragma unroll
                for (int side = 0; side < 2; ++side) {
                    if (!(any >> (16 * side) & 1)) continue;                             // warp-uniform
                    const int kv = __shfl_sync(0xffffffffu, h_now - a.nq, 16 * side);
                    const size_t grp = ((size_t)s_slot[r] * a.nkv + kv) * 4;
                    exl3::quant_x4(s_k[(hw & ~1) + side], a.qk + grp * a.k_bits, a.sk + grp, 4, a.k_bits);
                    exl3::quant_x4(a.v + ((size_t)row * a.nkv + kv) * 128, a.qv + grp * a.v_bits, a.sv + grp, 4, a.v_bits);
                }
                __syncwarp();
            }
        }
    }
}

}  // namespace

static_assert(sizeof(exl3_rope_append_args) == 15 * 8 + 16 * 4 + 64, "the bindings pack it without padding");

extern "C" int exl3_rope_append_paged(exl3_ctx* ctx, exl3_stream stream, const exl3_rope_append_args* r)
{
    EXL3_REQUIRE(ctx && r, "rope_append_paged: null argument");
    EXL3_REQUIRE(r->bsz >= 0 && r->seq >= 0 && r->rows >= 0 && r->nq >= 0 && r->nkv > 0 && r->pages > 0 && r->pages_per_seq > 0, "rope_append_paged: bad shape");
    const bool empty = r->bsz == 0 || r->seq == 0 || r->rows == 0, quant = r->k_bits != 0 || r->v_bits != 0;      // an empty call touches none of its tensors
    EXL3_REQUIRE(empty || (r->k && r->v && r->block_table && r->cache_seqlens && r->k_cache && r->v_cache && (!quant || (r->k_scales && r->v_scales))),
                 "rope_append_paged: null argument");
    EXL3_REQUIRE(r->q || r->nq == 0 || empty, "rope_append_paged: q is null but nq > 0");
    EXL3_REQUIRE(r->cu_q || (long long)r->bsz * r->seq == r->rows, "rope_append_paged: rows must be bsz * seq without cu_q");
    EXL3_REQUIRE(r->nq < (1 << 20) && r->nkv < (1 << 20), "rope_append_paged: too many heads");
    if (r->hd != 128) return exl3_fail(ctx, EXL3_ERR_UNSUPPORTED, "rope_append_paged: head_dim must be 128");
    EXL3_REQUIRE(!quant || (r->k_bits >= 2 && r->k_bits <= 8 && r->v_bits >= 2 && r->v_bits <= 8), "rope_append_paged: bits must be 2..8");
    EXL3_REQUIRE(r->rope_mode == EXL3_ROPE_NEOX || r->rope_mode == EXL3_ROPE_GPTJ || r->rope_mode == EXL3_ROPE_NONE, "rope_append_paged: unknown rope_mode");
    RopePagedArgs a = {(const half*)r->q, (half*)(r->out_q ? r->out_q : const_cast<void*>(r->q)), (const half*)r->k, (const half*)r->v, r->inv_freq, r->positions,
                       (const half*)r->q_norm, (const half*)r->k_norm, quant ? nullptr : (half*)r->k_cache, quant ? nullptr : (half*)r->v_cache,
                       quant ? (uint32_t*)r->k_cache : nullptr, (half*)r->k_scales, quant ? (uint32_t*)r->v_cache : nullptr, (half*)r->v_scales,
                       r->block_table, r->cache_seqlens, r->cu_q, r->norm_eps, r->norm_constant_bias, r->attn_factor, r->n_freq, r->rope_mode, r->bsz, r->seq,
                       r->rows, r->nq, r->nkv, r->pages, r->pages_per_seq, r->k_bits, r->v_bits, {}};
    if (r->rope_mode != EXL3_ROPE_NONE) {
        EXL3_REQUIRE(r->inv_freq, "rope_append_paged: null inv_freq");
        EXL3_REQUIRE(r->n_freq > 0 && 2 * r->n_freq <= r->hd, "rope_append_paged: 2*n_freq must be <= head_dim");
        if (r->rope_mode == EXL3_ROPE_NEOX && r->n_freq % 8 != 0)
            return exl3_fail(ctx, EXL3_ERR_UNSUPPORTED, "rope_append_paged: NEOX mode needs n_freq % 8 == 0");
        EXL3_REQUIRE(r->positions ? r->n_axes >= 1 : r->n_axes <= 1, "rope_append_paged: several axes need positions [n_axes, rows]");
        for (int f = 0; f < r->n_freq; ++f) {
            EXL3_REQUIRE(r->freq_axis[f] == 0 || r->freq_axis[f] < r->n_axes, "rope_append_paged: freq_axis names an axis that positions do not have");
            a.axis[f] = r->freq_axis[f];
        }
    }
    EXL3_REQUIRE(aligned16(r->q) && aligned16(r->out_q) && aligned16(r->k) && aligned16(r->v) && aligned16(r->q_norm) && aligned16(r->k_norm) &&
                 aligned16(r->k_cache) && aligned16(r->v_cache), "rope_append_paged: pointers must be 16-byte aligned");
    EXL3_REQUIRE(!quant || quant_planes_aligned(r->k_cache, r->k_scales, r->v_cache, r->v_scales), "rope_append_paged: scale planes must be 8-byte aligned");
    int dev = -1;
    EXL3_REQUIRE(cudaGetDevice(&dev) == cudaSuccess && dev == ctx->device, "rope_append_paged: the context's device must be the current one");
    if (empty) return EXL3_OK;
    const int heads = a.nq + a.nkv;
    // Eight rows per block share its start, a chain of loads and angles of about 3 us; where that leaves SMs idle, a row per block, its
    // heads over several blocks
    const bool many = a.rows >= RP_ROWS * 4 * ctx->num_sms;
    const dim3 grid(many ? (a.rows + RP_ROWS - 1) / RP_ROWS : a.rows,
                    many ? 1 : (unsigned)max(1, min((heads + RP_HALF - 1) / RP_HALF, 4 * ctx->num_sms / a.rows)));
    cudaStream_t st = (cudaStream_t)stream;
    if (quant) {
        if (many) exl3_launch_first(ctx, rope_paged_kernel<RP_ROWS, 2, true>, grid, RP_THREADS, 0, st, a);
        else exl3_launch_first(ctx, rope_paged_kernel<1, 1, true>, grid, RP_THREADS, 0, st, a);
    } else {
        if (many) exl3_launch_first(ctx, rope_paged_kernel<RP_ROWS, 2, false>, grid, RP_THREADS, 0, st, a);
        else exl3_launch_first(ctx, rope_paged_kernel<1, 1, false>, grid, RP_THREADS, 0, st, a);
    }
    ctx->launches++;
    return exl3_check_launch(ctx, "rope_append_paged");
}
