// How the attention over the paged cache is cut into work: shared by its kernels and by the kernel that joins their
// partial results.
//
// A request's query rows, heads of a kv head's group packed beside one another (row = token * group + head in group),
// are cut into row tiles; an item is one row tile of one kv head, and its work is the tiles of `kTokens` cached tokens
// that any of its rows sees (one unit for an item that sees nothing: its zeros have to be written).  The units of all
// items, request by request, head by head, row tile by row tile, are numbered through and dealt to the blocks in equal
// contiguous chunks, so lengths need not be known on the host and a long request costs no more than the same tokens in
// short ones.  An item inside one chunk is finished there; the pieces of any other leave float32 partial results
// (unnormalised output, running maximum and sum), which the joining kernel adds in the order of the chunks: the result
// is the same from run to run.
#pragma once

#include <cstdint>

#include "cache.h"
#include "ptx.cuh"

namespace blaze {

constexpr int kAttnMaxRequests = 8192;

// What the joining kernel has to know of an item that lies in more than one chunk.
struct AttnCut {
    int first, last;                  // its first and last block; first = -1: nothing is cut here
    int inside;                       // 1: its first piece starts inside the first block's chunk
    int q0, head, row0, rows, pad;
};

struct CacheAttentionParams {
    int requests, tokens, heads, kv_heads, group;
    int block_shift, num_blocks, max_blocks;
    int max_q, max_kv;
    int causal, window;
    float scale_log2;                 // scale * log2(e)
    const void* q;
    long long q_token_stride, q_head_stride;
    void* out;
    long long out_token_stride, out_head_stride;
    float* lse;
    const int* row_offsets;
    const int* kv_len;
    const int* table;
    long long table_stride;
    const float* k_scale;
    const float* v_scale;
    long long scale_stride;
    int few_rows;                     // requests of at most so many packed rows go to the few-rows kernel, others not
    int take_few, take_many;          // which of the two this launch takes
    int min_chunk;                    // units per block, at least
    float* part_out;                  // [block][2][row tile][head_dim]
    float* part_ml;                   // [block][2][row tile][2]
    struct AttnCut* cuts;             // [block]: the item that the end of the block's chunk cuts
    int* status;
};

// Bounded wait of a whole warp.
__device__ __forceinline__ bool attn_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    long long t0 = 0;
    for (;;) {
        const bool ok = mbar_try_wait(bar, parity);
        if (__all_sync(0xffffffffu, ok)) return true;
        const long long now = clock64();
        if (t0 == 0) t0 = now;
        int over = *abort_flag;
        if (now - t0 > BLAZE_WAIT_LIMIT_CYCLES) {
            over = 1;
            *abort_flag = 1;
            atomicCAS(status, 0, code);
        }
        if (__any_sync(0xffffffffu, over != 0)) return false;
    }
}

struct AttnRequest {
    int q0, qlen, kv;
};

__device__ __forceinline__ AttnRequest attn_request(const CacheAttentionParams& p, int r) {
    AttnRequest q;
    const int a = min(max(p.row_offsets[r], 0), p.tokens);
    const int b = min(max(p.row_offsets[r + 1], a), p.tokens);
    q.q0 = a;
    q.qlen = min(b - a, p.max_q);
    q.kv = min(max(p.kv_len[r], 0), p.max_kv);
    const bool few = (long long)q.qlen * p.group <= p.few_rows;
    if (few ? !p.take_few : !p.take_many) q.qlen = 0;
    return q;
}

// Tokens [lo, hi) that the rows of row tile `qt` see between them.
template <int kRows>
__device__ __forceinline__ void attn_span(const CacheAttentionParams& p, const AttnRequest& q, int qt, int& lo, int& hi) {
    const int rows = q.qlen * p.group;
    const int i0 = (qt * kRows) / p.group;
    const int i1 = (min(rows, (qt + 1) * kRows) - 1) / p.group;
    const int off = q.kv - q.qlen;
    hi = p.causal ? min(q.kv, off + i1 + 1) : q.kv;
    lo = p.window > 0 ? max(0, off + i0 - p.window + 1) : 0;
    if (hi <= lo) { lo = 0; hi = 0; }
}

template <int kTokens>
__device__ __forceinline__ int attn_units(int lo, int hi) {
    return hi <= lo ? 1 : (hi + kTokens - 1) / kTokens - lo / kTokens;
}

// Units of row tile t.
template <int kRows, int kTokens>
__device__ __forceinline__ int attn_units_of_tile(const CacheAttentionParams& p, const AttnRequest& q, int t) {
    int lo, hi;
    attn_span<kRows>(p, q, t, lo, hi);
    return attn_units<kTokens>(lo, hi);
}

// prefix[r] = units before request r, prefix[requests] = all of them.  Called by the whole block.
template <int kRows, int kTokens>
__device__ __forceinline__ void attn_prefix(const CacheAttentionParams& p, int* prefix, int* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int carry = 0;
#pragma unroll 1
    for (int base = 0; base < p.requests; base += blockDim.x) {
        const int r = base + threadIdx.x;
        AttnRequest q = {0, 0, 0};
        if (r < p.requests) q = attn_request(p, r);
        const int tiles = (q.qlen * p.group + kRows - 1) / kRows;
        int u = tiles > 0 ? attn_units_of_tile<kRows, kTokens>(p, q, 0) : 0;
        // requests of many row tiles: the warp's lanes share them
        uint32_t many = __ballot_sync(0xffffffffu, tiles > 1);
        while (many) {
            const int src = __ffs(many) - 1;
            many &= many - 1;
            AttnRequest o;
            o.q0 = 0;
            o.qlen = __shfl_sync(0xffffffffu, q.qlen, src);
            o.kv = __shfl_sync(0xffffffffu, q.kv, src);
            const int n = __shfl_sync(0xffffffffu, tiles, src);
            int sum = 0;
#pragma unroll 1
            for (int t = lane; t < n; t += 32) sum += attn_units_of_tile<kRows, kTokens>(p, o, t);
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == src) u = sum;
        }
        u *= p.kv_heads;
        int inc = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) warp_sums[warp] = inc;
        __syncthreads();
        int before = carry, total = carry;
#pragma unroll 1
        for (int w = 0; w < warps; ++w) {
            const int s = warp_sums[w];
            if (w < warp) before += s;
            total += s;
        }
        if (r < p.requests) prefix[r] = before + inc - u;
        carry = total;
        __syncthreads();
    }
    if (threadIdx.x == 0) prefix[p.requests] = carry;
    __syncthreads();
}

// Units of a block's chunk: equal for all blocks but the last that has any.
__device__ __forceinline__ int attn_chunk(const CacheAttentionParams& p, int total, int blocks) {
    return max((total + blocks - 1) / blocks, p.min_chunk);
}

// The piece of an item that starts at unit u and ends at the item's end or at unit `end`; called by whole warps.
struct AttnPiece {
    AttnRequest req;
    int r, head, row0, rows;          // first packed row of the tile, packed rows of the request
    int lo, hi;                       // tokens that the whole item's rows see between them
    int tile0, tile1;                 // tiles of this piece
    int item0, item1;                 // units of the item
};

template <int kRows, int kTokens>
__device__ __forceinline__ AttnPiece attn_piece(const CacheAttentionParams& p, const int* prefix, int u, int end) {
    AttnPiece s;
    int a = 0, b = p.requests;
#pragma unroll 1
    while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (prefix[mid] <= u) a = mid; else b = mid;
    }
    s.r = a;
    s.req = attn_request(p, a);
    s.rows = s.req.qlen * p.group;
    const int per_head = (prefix[a + 1] - prefix[a]) / p.kv_heads;
    const int local = u - prefix[a];
    s.head = local / per_head;
    int rem = local - s.head * per_head;
    int qt = 0;
    if (s.rows > kRows) {
        // the row tile that unit `rem` of the head lies in: the warp's lanes sum the tiles' units 32 at a time
        const int lane = threadIdx.x & 31, tiles = (s.rows + kRows - 1) / kRows;
#pragma unroll 1
        for (;; qt += 32) {
            const int n = qt + lane < tiles ? attn_units_of_tile<kRows, kTokens>(p, s.req, qt + lane) : 0x3FFFFFFF;
            int inc = min(n, 0x3FFFFFFF);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc = min(inc + y, 0x3FFFFFFF);
            }
            const uint32_t beyond = __ballot_sync(0xffffffffu, inc > rem);
            if (beyond) {
                const int at = __ffs(beyond) - 1;
                if (at > 0) rem -= __shfl_sync(0xffffffffu, inc, at - 1);
                qt += at;
                break;
            }
            rem -= __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    attn_span<kRows>(p, s.req, qt, s.lo, s.hi);
    const int n = attn_units<kTokens>(s.lo, s.hi);
    s.row0 = qt * kRows;
    s.item0 = u - rem;
    s.item1 = s.item0 + n;
    const int take = min(s.item1, end) - u;
    s.tile0 = s.lo / kTokens + rem;
    s.tile1 = s.hi <= s.lo ? s.tile0 : s.tile0 + take;
    return s;
}
// The cut at the end of block `block`'s chunk, s being the chunk's last piece.
__device__ __forceinline__ void attn_write_cut(const CacheAttentionParams& p, const AttnPiece& s, int block, int chunk, int end) {
    AttnCut c;
    c.first = s.item1 > end ? s.item0 / chunk : -1;
    c.last = (s.item1 - 1) / chunk;
    c.inside = s.item0 != c.first * chunk ? 1 : 0;
    c.q0 = s.req.q0;
    c.head = s.head;
    c.row0 = s.row0;
    c.rows = s.rows;
    c.pad = 0;
    p.cuts[block] = c;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Without flushing: 1 / v_scale is subnormal for a scale above 2^126.
__device__ __forceinline__ float ex2_subnormal(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two E4M3 codes (the low or the high half of w) as two halves.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// One box of a page: `row` and on of (head, block).
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int head, int block) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(row), "r"(head), "r"(block)
        : "memory");
}

// A V scale enters the exponent; below 2^-64 (which the store never writes) it counts as that, so that a sum of p / v_scale
// stays far below float32's end.  A token's p vanishes from the sum when its score (in powers of two, with its V scale) is
// 2^138 below the row's largest: with V scales at most 2^96 apart, a weight of 2^-42 of the largest one's.
constexpr float kMinLogScale = -64.0f;

// Power of two that brings the largest magnitude of a row of bf16 queries to [2^14, 2^15), so that the row fits half
// with all its bits; 1 for half queries, which are taken as they are.
__device__ __forceinline__ int query_shift(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23) - 127;
    return amax > 0.0f ? min(max(14 - e, -120), 120) : 0;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <bool kBf16>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
    return kBf16 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
}

}  // namespace blaze
