// The many-rows kernel of the attention over the paged cache (prompts and chunks of prompts): both products on the
// tensor cores with tcgen05 (kind::f16, float32 accumulation).  The formulas are at the top of cache_attention.cu.
//
// A row tile is 256 packed query rows, two sub-tiles A and B of 128, one accumulator row per thread of a warpgroup each;
// a tile of the cache is 128 tokens.  Roles:
//   warps 0-3, 4-7   softmax of sub-tile A / B: scores from TMEM, probabilities back into the same TMEM columns as half
//                    (the A operand of P V), O re-scaled in TMEM when a row's maximum has grown by more than 2^3
//                    since it was last taken, the piece's epilogue
//   warps 8-11       codes -> half: expand (exactly) the codes of an operand tile out of its staging slot into the
//                    128-byte-swizzled operand tile, a ring of three that K and V take turns in
//   warp 12          issues the MMAs: P_A V(t), Q_A K(t+1), P_B V(t), Q_B K(t+1), so each warpgroup's softmax runs while the
//                    tensor cores work for the other one
//   warp 13          fetches the pages' codes into the staging slots by TMA, an operand tile and a half ahead; block numbers
//                    and scales of the tiles
// The softmax threads also bring their own query row into shared memory at the start of a piece.
// Q K^T takes K as the K-major operand; P V takes V as it lies, dims contiguous (MN-major), no transposition anywhere.
// 769 rows of 16 heads of 128 on 15k and 30k tokens: 221 us, 720 TFLOP/s, tensor pipe and exponentials 37 % busy each; 4 prompts
// of up to 4096 rows of 32 heads: 625 us, 450 TFLOP/s.  Bound, within a piece, by the chain of a sub-tile: softmax, hand-over to the
// issuing warp, MMAs, hand-over back, which the other sub-tile's fills only partly (2.9 us per 128 tokens); between pieces
// by the epilogue and the next queries, one behind the other (10 us a piece in the prompts, whose blocks have equal tiles but
// up to 25 pieces: they end after 335 to 619 us).  Spills at the 128 registers that ptxas allocates for: 44 to 52 bytes stored
// for heads of 128, 16 for heads of 64.
#pragma once

#include "cache_schedule.cuh"

namespace blaze {

constexpr int kManyRows = 256;
constexpr int kManyTokens = 128;
constexpr int kManyThreads = 32 * 16;      // warps 14, 15 only complete the last warpgroup
// Registers of a thread of the softmax, converting and issuing warpgroups (a softmax thread holds 64 to 96 scores);
// the launch has 128 each, 512 for the four.
constexpr int kSoftmaxRegs = 176, kConvertRegs = 88, kIssueRegs = 72;
constexpr int kManyLaunchRegs = 128;
static_assert(2 * kSoftmaxRegs + kConvertRegs + kIssueRegs <= 4 * kManyLaunchRegs, "setmaxnreg draws on what the launch has");
constexpr int kManyMeta = 4;              // tiles whose scales are held

// A row's reference is set 2^12 below its largest score (with the V scale in it) and kept until a score passes it by 2^15
// (half ends at 2^16).  So the largest probability of a row is held as 2^12 to 2^15: in half the values down to 2^-26 of it
// have all their 11 bits, smaller ones are off by at most 2^-37 of it and vanish below that, while the sum l counts them in
// full.  A row's output may rest on such values, where the heaviest token has no value (an attention sink).  A reference 2^3
// below the largest leaves 2^-17 and 2^-28 (2.4 % off at weights of 2^-24.5).
constexpr float kManyShift = 12.0f;
constexpr float kManyGrow = 15.0f;

template <int kDim>
struct ManySmem {
    static constexpr int kHalves = kDim / 64;                        // 64-wide (128-byte) column halves
    static constexpr int kOperandBytes = 128 * kDim * 2;             // 128 rows of Q, K or V as half
    static constexpr int kQOffset = 0;                               // A, B
    static constexpr int kRingOffset = 2 * kOperandBytes;            // three operand tiles, K and V in turn
    static constexpr int kRawOffset = kRingOffset + 3 * kOperandBytes;     // codes of a K and of a V tile
    static constexpr int kRawBytes = 128 * kDim;
    static constexpr int kMetaOffset = kRawOffset + 2 * kRawBytes;   // float4 [kManyMeta][8]
    static constexpr int kBarOffset = kMetaOffset + kManyMeta * 8 * 16;
    static constexpr int kNumBars = 2 + 6 + kManyMeta + 6 + 4;
    static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
    static constexpr int kPrefixOffset = kMiscOffset + 128;
    static int bytes(int requests) { return 1024 + kPrefixOffset + (requests + 1) * 4; }
};

// Operand of kDim or 128 columns stored [k row][64 columns] per half with the 128-byte swizzle, the contiguous
// direction being the instruction's N: halves `half_bytes` apart, groups of 8 k rows 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t smem_addr, uint32_t half_bytes) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(half_bytes >> 4) << 16;               // leading byte offset: next 64 columns
    d |= static_cast<uint64_t>(1024 >> 4) << 32;                     // stride byte offset: next 8 k rows
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

__host__ __device__ constexpr uint32_t umma_idesc_half(uint32_t n, bool b_mn) {          // M = 128, half x half -> float32
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
template <int kRegs>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// O of this warp's 32 rows times a factor per row.
template <int kDim>
__device__ __forceinline__ void rescale(uint32_t to, float al) {
#pragma unroll 1
    for (int c = 0; c < kDim / 16; ++c) {
        uint32_t v[16];
        tmem_ld_32x16(to + c * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * al);
        tmem_st_32x16(to + c * 16, v);
    }
}

// Tokens [lo, hi) that any row of the sub-tile of 128 rows at `row0` sees, and [all_lo, all_hi) that every row sees.
struct SubTile {
    int lo, hi, all_lo, all_hi;
    __device__ __forceinline__ bool active(int t) const {
        return t * kManyTokens < hi && (t + 1) * kManyTokens > lo;
    }
    __device__ __forceinline__ bool masked(int t) const {
        return t * kManyTokens < all_lo || (t + 1) * kManyTokens > all_hi;
    }
};
__device__ __forceinline__ SubTile sub_tile(const CacheAttentionParams& p, const AttnPiece& s, int row0, int row1) {
    SubTile x;
    const int end = min(s.rows, row1);
    if (row0 >= end) {
        x.lo = x.hi = x.all_lo = x.all_hi = 0;
        return x;
    }
    const int i0 = row0 / p.group, i1 = (end - 1) / p.group, off = s.req.kv - s.req.qlen;
    x.hi = p.causal ? min(s.req.kv, off + i1 + 1) : s.req.kv;
    x.lo = p.window > 0 ? max(0, off + i0 - p.window + 1) : 0;
    x.all_hi = p.causal ? min(s.req.kv, off + i0 + 1) : s.req.kv;
    x.all_lo = p.window > 0 ? max(0, off + i1 - p.window + 1) : 0;
    if (x.hi <= x.lo) x.lo = x.hi = 0;
    return x;
}

// 16 E4M3 codes -> 16 halves.
__device__ __forceinline__ void codes_to_half(const uint4& w, uint4& a, uint4& b) {
    a = make_uint4(codes_lo(w.x), codes_hi(w.x), codes_lo(w.y), codes_hi(w.y));
    b = make_uint4(codes_lo(w.z), codes_hi(w.z), codes_lo(w.w), codes_hi(w.w));
}

template <int kDim, bool kBf16>
__global__ void __launch_bounds__(kManyThreads, 1)
cache_attention_many_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                            const CacheAttentionParams p, const CacheView cache) {
    using L = ManySmem<kDim>;
    extern __shared__ uint8_t many_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(many_smem_raw) + 1023) & ~uintptr_t(1023));
    float4* meta = reinterpret_cast<float4*>(smem + L::kMetaOffset);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOffset);
    uint64_t* q_full = bars;                  // the softmax warps
    uint64_t* q_free = bars + 1;              // the last Q K^T of the piece
    uint64_t* full = bars + 2;                // [3] operand tile expanded (the converting warps)
    uint64_t* free_ = bars + 5;               // [3] its last product done
    uint64_t* meta_full = bars + 8;           // [kManyMeta]
    uint64_t* s_full = meta_full + kManyMeta; // [2] sub-tiles
    uint64_t* p_full = s_full + 2;            // [2]
    uint64_t* pv_done = s_full + 4;           // [2]
    uint64_t* raw_full = s_full + 6;          // [2] codes of a K tile, of a V tile are there
    uint64_t* raw_free = s_full + 8;          // [2] they have been read (the converting warps)
    int* misc = reinterpret_cast<int*>(smem + L::kMiscOffset);           // [0, 16): sums; 16: TMEM; 17: abort; 18..25: NaN tiles
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + 16);
    volatile int* abort_flag = misc + 17;
    volatile int* nan_tile = misc + 18;       // number (+ 1) of the last tile of each 8 whose V lost NaN codes
    int* prefix = reinterpret_cast<int*>(smem + L::kPrefixOffset);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 8);
        mbar_init(q_free, 1);
        for (int i = 0; i < 3; ++i) {
            mbar_init(&full[i], 4);
            mbar_init(&free_[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_free[i], 4);
        }
        for (int i = 0; i < kManyMeta; ++i) mbar_init(&meta_full[i], 1);
        *abort_flag = 0;
        for (int i = 0; i < 8; ++i) nan_tile[i] = 0;
        fence_mbar_init();
    }
    if (warp == 12) tmem_alloc<1>(tmem_slot, 512);
    grid_dependency_wait();
    tcgen05_fence_before();
    attn_prefix<kManyRows, kManyTokens>(p, prefix, misc);
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_s[2] = {tmem, tmem + 128};
    const uint32_t tmem_o[2] = {tmem + 256, tmem + 256 + kDim};
    const int total = prefix[p.requests];
    const int chunk = attn_chunk(p, total, gridDim.x);
    const long long begin64 = (long long)blockIdx.x * chunk;
    const int begin = (int)min(begin64, (long long)total);
    const int end = (int)min(begin64 + chunk, (long long)total);
    bool ok = true;
    if (threadIdx.x == 0) p.cuts[blockIdx.x].first = -1;          // until this thread knows better

    if (warp < 8) {
        // ------------------------------------------------------------------ softmax
        regs_inc<kSoftmaxRegs>();
        const int x = warp >> 2;                              // sub-tile
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem_s[x] + lanes, to = tmem_o[x] + lanes;
        const int row_in_tile = x * 128 + (warp & 3) * 32 + lane;
        int n_piece = 0, n_tile = 0, n_mine = 0;              // pieces, tiles of the block, tiles of this sub-tile so far
        for (int u = begin; u < end && ok; ++n_piece) {
            const AttnPiece s = attn_piece<kManyRows, kManyTokens>(p, prefix, u, end);
            const int u_next = u + max(1, s.tile1 - s.tile0);
            const SubTile sub = sub_tile(p, s, s.row0 + x * 128, s.row0 + x * 128 + 128);
            const int row = s.row0 + row_in_tile;
            const bool there = row < s.rows;
            const int i = there ? row / p.group : 0;
            const int head = s.head * p.group + (there ? row - i * p.group : 0);
            const int pos = s.req.kv - s.req.qlen + i;
            const int see_hi = there ? (p.causal ? min(s.req.kv, pos + 1) : s.req.kv) : 0;
            const int see_lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
            // ---- this thread's query row, as half (bf16 rows scaled by a power of two, the sign of `scale` taken in)
            float factor = 1.0f;
            {
                constexpr int kLoads = kDim / 8;
                uint4 w[kLoads];
                const uint16_t* src = static_cast<const uint16_t*>(p.q) + (long long)(s.req.q0 + i) * p.q_token_stride +
                                      (long long)head * p.q_head_stride;
#pragma unroll
                for (int k = 0; k < kLoads; ++k)
                    w[k] = there ? *reinterpret_cast<const uint4*>(src + 8 * k) : make_uint4(0, 0, 0, 0);
                if constexpr (kBf16) {
                    uint32_t mag = 0;
#pragma unroll
                    for (int k = 0; k < kLoads; ++k) {
                        const uint32_t* e = &w[k].x;
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const uint32_t a = e[h] & 0x7FFFu, b = (e[h] >> 16) & 0x7FFFu;
                            mag = max(mag, max(a < 0x7F80u ? a : 0u, b < 0x7F80u ? b : 0u));
                        }
                    }
                    const int shift = query_shift(__uint_as_float(mag << 16));
                    factor = pow2i(-shift);
                    const float mul = p.scale_log2 < 0.0f ? -pow2i(shift) : pow2i(shift);
#pragma unroll
                    for (int k = 0; k < kLoads; ++k) {
                        uint32_t* e = &w[k].x;
#pragma unroll
                        for (int h = 0; h < 4; ++h)
                            e[h] = pack_f16(__uint_as_float(e[h] << 16) * mul, __uint_as_float(e[h] & 0xFFFF0000u) * mul);
                    }
                } else {
                    const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
                    for (int k = 0; k < kLoads; ++k) {
                        w[k].x ^= flip; w[k].y ^= flip; w[k].z ^= flip; w[k].w ^= flip;
                    }
                }
                if (n_piece > 0) {
                    ok = attn_wait(q_free, (n_piece - 1) & 1, abort_flag, p.status, DEV_TIMEOUT_SMEM_EMPTY);
                    if (!ok) break;
                }
                uint8_t* at = smem + L::kQOffset + x * L::kOperandBytes + (row_in_tile & 127) * 128;
#pragma unroll
                for (int k = 0; k < kLoads; ++k)
                    *reinterpret_cast<uint4*>(at + (k >> 3) * 16384 + (((k & 7) ^ (row_in_tile & 7)) << 4)) = w[k];
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }

            float m = -INFINITY, l = 0.0f;
            int done = 0;                                     // tiles of this piece whose P V has been asked for
            bool nans = false;                                // V of one of them lost NaN codes
            int before = 0;                                   // number of the last of them
            for (int t = s.tile0; t < s.tile1; ++t, ++n_tile) {
                if (!sub.active(t)) continue;
                ok = attn_wait(&meta_full[n_tile % kManyMeta], (n_tile / kManyMeta) & 1, abort_flag, p.status, DEV_TIMEOUT_SMEM_FULL) &&
                     attn_wait(&s_full[x], n_mine & 1, abort_flag, p.status, DEV_TIMEOUT_TMEM_FULL);
                if (!ok) break;
                tcgen05_fence_after();
                if (done > 0) nans |= nan_tile[before & 7] == before + 1;
                const float4* mt = meta + (n_tile % kManyMeta) * 8;
                const bool masked = sub.masked(t);
                const int tok0 = t * kManyTokens;
                float ms = 0.0f;
                // A new reference, only where a score has outgrown the old one by 2^15 (and in a piece's first tile).
                auto refer = [&](float mx) {
                    const bool grow = mx > m + kManyGrow;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float m_new = grow ? mx - kManyShift : m;
                        const float al = grow ? (m == -INFINITY ? 0.0f : ex2(m - m_new)) : 1.0f;
                        m = m_new;
                        l *= al;
                        if (done > 0) {
                            ok = attn_wait(&pv_done[x], (n_mine - 1) & 1, abort_flag, p.status, DEV_TIMEOUT_TMEM_FULL);
                            tcgen05_fence_after();
                            rescale<kDim>(to, al);
                        }
                    }
                    ms = m == -INFINITY ? 0.0f : m;
                };
                // Probabilities of 32 tokens, over the scores' own columns (they fit those of 16 tokens, read before).
                auto exponentials = [&](int c, const uint32_t (&v)[32], float floor_k1) {
                    uint32_t w[16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float4 q = mt[2 * c + h];
                        const float k1 = fmaxf(factor * q.x, floor_k1), k0 = q.y - ms;
                        float part = 0.0f, part2 = 0.0f;
#pragma unroll
                        for (int k = 0; k < 16; k += 4) {
                            const float a = ex2(fmaf(__uint_as_float(v[16 * h + k]), k1, k0));
                            const float b = ex2(fmaf(__uint_as_float(v[16 * h + k + 1]), k1, k0));
                            const float d = ex2(fmaf(__uint_as_float(v[16 * h + k + 2]), k1, k0));
                            const float e = ex2(fmaf(__uint_as_float(v[16 * h + k + 3]), k1, k0));
                            part += a + b;
                            part2 += d + e;
                            w[8 * h + (k >> 1)] = pack_f16(a, b);
                            w[8 * h + (k >> 1) + 1] = pack_f16(d, e);
                        }
                        l = fmaf(part + part2, q.z, l);
                    }
                    tmem_st_32x16(ts + c * 16, w);
                };
                // (blocks that do not exist have codes of zero and an exponent of -inf)
                float mx = -INFINITY;
                if (!masked) {
                    // the largest of the scores of 64..127 first, then of 0..63, which stay for the exponentials; the others
                    // are read again behind them
                    uint32_t sc[2][32];
                    auto largest = [&](int c, const uint32_t (&v)[32]) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float4 q = mt[2 * c + h];
                            const uint32_t* e = &v[16 * h];
                            float a = __uint_as_float(e[0]), b = __uint_as_float(e[1]);
#pragma unroll
                            for (int k = 2; k < 14; k += 4) {
                                a = max3(a, __uint_as_float(e[k]), __uint_as_float(e[k + 1]));
                                b = max3(b, __uint_as_float(e[k + 2]), __uint_as_float(e[k + 3]));
                            }
                            a = max3(a, __uint_as_float(e[14]), __uint_as_float(e[15]));
                            mx = fmaxf(mx, fmaf(fmaxf(a, b), factor * q.x, q.y));
                        }
                    };
                    tmem_ld_32x32(ts + 64, sc[0]);
                    tmem_ld_32x32(ts + 96, sc[1]);
                    tmem_ld_wait();
                    largest(2, sc[0]);
                    largest(3, sc[1]);
                    tmem_ld_32x32(ts, sc[0]);
                    tmem_ld_32x32(ts + 32, sc[1]);
                    tmem_ld_wait();
                    largest(0, sc[0]);
                    largest(1, sc[1]);
                    refer(mx);
                    if (!ok) break;
                    exponentials(0, sc[0], 0.0f);
                    tmem_ld_32x32(ts + 64, sc[0]);
                    exponentials(1, sc[1], 0.0f);
                    tmem_ld_wait();
                    tmem_ld_32x32(ts + 96, sc[1]);
                    exponentials(2, sc[0], 0.0f);
                    tmem_ld_wait();
                    exponentials(3, sc[1], 0.0f);
                } else {
                    // bits of the tokens of 32 columns that this row sees
                    auto seen = [&](int c) -> uint32_t {
                        const int a = max(see_lo - (tok0 + 32 * c), 0), b = min(see_hi - (tok0 + 32 * c), 32);
                        return b > a ? (0xFFFFFFFFu >> (32 - b)) & (0xFFFFFFFFu << a) : 0u;
                    };
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t v[32];
                        __syncwarp();
                        tmem_ld_32x32(ts + c * 32, v);
                        tmem_ld_wait();
                        const uint32_t bits = seen(c);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float4 q = mt[2 * c + h];
                            float g = -INFINITY;
#pragma unroll
                            for (int k = 16 * h; k < 16 * h + 16; ++k) g = fmaxf(g, bits >> k & 1 ? __uint_as_float(v[k]) : -INFINITY);
                            if (bits >> (16 * h) & 0xFFFFu) mx = fmaxf(mx, fmaf(g, factor * q.x, q.y));
                        }
                    }
                    __syncwarp();
                    refer(mx);
                    if (!ok) break;
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t v[32];
                        __syncwarp();
                        tmem_ld_32x32(ts + c * 32, v);
                        tmem_ld_wait();
                        // a score that the row does not see may be anything: taken out before the exponential (whose
                        // factor then must not be zero)
                        const uint32_t bits = seen(c);
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[k] = bits >> k & 1 ? v[k] : 0xFF800000u;
                        exponentials(c, v, 1e-37f);
                    }
                }
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[x]);
                before = n_tile;
                ++done;
                ++n_mine;
            }
            if (!ok) break;
            // ---- epilogue
            if (done > 0) {
                ok = attn_wait(&pv_done[x], (n_mine - 1) & 1, abort_flag, p.status, DEV_TIMEOUT_TMEM_FULL);
                if (!ok) break;
                tcgen05_fence_after();
                nans |= nan_tile[before & 7] == before + 1;
            }
            const bool whole = s.item0 >= begin && s.item1 <= end;
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            const long long slot = (long long)blockIdx.x * 2 + (u == begin ? 0 : 1);
            uint16_t* out = static_cast<uint16_t*>(p.out) + (long long)(s.req.q0 + i) * p.out_token_stride +
                            (long long)head * p.out_head_stride;
            float* part = p.part_out + (slot * kManyRows + row_in_tile) * kDim;
#pragma unroll 1
            for (int c = 0; c < kDim / 32; ++c) {
                uint32_t v[32];
                __syncwarp();
                if (done > 0) {
                    tmem_ld_32x32(to + c * 32, v);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] = 0;
                }
                if (nans && there) {
                    // NaN codes of V in tiles that not every row sees were taken out of the product: the rows that do see
                    // them get their NaN here, from the codes themselves
                    const SubTile all = sub_tile(p, s, s.row0, s.row0 + kManyRows);
                    for (int t = s.tile0; t < s.tile1; ++t) {
                        if (!all.masked(t)) continue;
                        const int a = max(see_lo, t * kManyTokens), b = min(see_hi, (t + 1) * kManyTokens);
                        for (int tok = a; tok < b; ++tok) {
                            const int block = p.table[(long long)s.r * p.table_stride + (tok >> p.block_shift)];
                            if (block < 0 || block >= p.num_blocks) continue;
                            const uint8_t* code = cache.v + block * cache.block_stride + s.head * cache.head_stride +
                                                  (long long)(tok & (cache.block_size - 1)) * cache.token_stride + c * 32;
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                if ((code[k] & 0x7F) == 0x7F) v[k] = 0x7FC00000u;
                        }
                    }
                }
                if (!there) {
                } else if (whole) {
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        uint4 w;
                        w.x = pack_out<kBf16>(__uint_as_float(v[k]) * inv, __uint_as_float(v[k + 1]) * inv);
                        w.y = pack_out<kBf16>(__uint_as_float(v[k + 2]) * inv, __uint_as_float(v[k + 3]) * inv);
                        w.z = pack_out<kBf16>(__uint_as_float(v[k + 4]) * inv, __uint_as_float(v[k + 5]) * inv);
                        w.w = pack_out<kBf16>(__uint_as_float(v[k + 6]) * inv, __uint_as_float(v[k + 7]) * inv);
                        *reinterpret_cast<uint4*>(out + c * 32 + k) = w;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<uint4*>(part + c * 32 + k) = make_uint4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                }
            }
            if (there) {
                if (whole) {
                    if (p.lse) p.lse[(long long)(s.req.q0 + i) * p.heads + head] = l != 0.0f ? (m + lg2(l)) * 0.6931471805599453f : -INFINITY;
                } else {
                    *reinterpret_cast<float2*>(p.part_ml + (slot * kManyRows + row_in_tile) * 2) = make_float2(m, l);
                }
            }
            if (threadIdx.x == 0 && u_next >= end) attn_write_cut(p, s, blockIdx.x, chunk, end);
            tcgen05_fence_before();                           // O has been read: the next piece may overwrite it
            __syncwarp();
            u = u_next;
        }
    } else if (warp < 12) {
        // ------------------------------------------------------------------ codes -> half
        regs_dec<kConvertRegs>();
        const int tid = threadIdx.x - 256;
        constexpr int kChunks = kDim / 16;                    // 16-code chunks of a row
        constexpr int kPasses = kDim / 16;                    // rows of a tile that a thread has a chunk of
        constexpr int kPassRows = 128 / kPasses;              // (16 or 32, multiples of the swizzles' eight rows)
        const int ch = tid % kChunks, r0 = tid / kChunks;
        // where a chunk's codes are in the staging slot, and where the two halves of what they become go, in an order that
        // keeps the eight lanes of a row on different banks
        const uint32_t raw_at = r0 * kDim + ((kDim == 128 ? ch ^ (r0 & 7) : ch ^ ((r0 >> 1) & 3)) << 4);
        const int flip = (ch >> 2) & 1;
        const uint32_t to_a = (ch >> 2) * 16384 + r0 * 128 + ((((ch & 3) * 2 + flip) ^ (r0 & 7)) << 4);
        const uint32_t to_b = (ch >> 2) * 16384 + r0 * 128 + ((((ch & 3) * 2 + 1 - flip) ^ (r0 & 7)) << 4);
        int n_tile = 0, ring = 0;                             // tiles so far; place in the ring
        uint32_t ring_phase = 1;
        for (int u = begin; u < end && ok;) {
            const AttnPiece s = attn_piece<kManyRows, kManyTokens>(p, prefix, u, end);
            u += max(1, s.tile1 - s.tile0);
            const SubTile all = sub_tile(p, s, s.row0, s.row0 + kManyRows);
            for (int t = s.tile0; t < s.tile1 && ok; ++t, ++n_tile) {
                const bool masked = all.masked(t);
#pragma unroll 1
                for (int which = 0; which < 2; ++which) {
                    ok = attn_wait(&raw_full[which], n_tile & 1, abort_flag, p.status, DEV_TIMEOUT_SMEM_FULL);
                    if (!ok) break;
                    const uint8_t* raw = smem + L::kRawOffset + which * L::kRawBytes + raw_at;
                    uint4 w[kPasses];
#pragma unroll
                    for (int j = 0; j < kPasses; ++j) w[j] = *reinterpret_cast<const uint4*>(raw + j * kPassRows * kDim);
                    // groups of 16 tokens that have been fetched
                    const uint32_t there = __float_as_uint(meta[(n_tile % kManyMeta) * 8].w);
                    if (masked || there != 0xFFu) {
                        // zeros in place of tokens that no row sees or that there are not and, of V, of NaN codes
                        bool any = false;
#pragma unroll
                        for (int j = 0; j < kPasses; ++j) {
                            const int row = j * kPassRows + r0, tok = t * kManyTokens + row;
                            if (tok < s.lo || tok >= s.hi || !(there >> (row >> 4) & 1)) w[j] = make_uint4(0, 0, 0, 0);
                            if (which == 1 && masked) {
                                uint32_t* e = &w[j].x;
#pragma unroll
                                for (int h = 0; h < 4; ++h) {
                                    const uint32_t nb = __vcmpeq4(e[h] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
                                    any |= nb != 0;
                                    e[h] &= ~nb;
                                }
                            }
                        }
                        if (any) nan_tile[n_tile & 7] = n_tile + 1;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&raw_free[which]);
                    ok = attn_wait(&free_[ring], ring_phase, abort_flag, p.status, DEV_TIMEOUT_SMEM_EMPTY);
                    if (!ok) break;
                    uint8_t* tile = smem + L::kRingOffset + ring * L::kOperandBytes;
#pragma unroll
                    for (int j = 0; j < kPasses; ++j) {
                        uint4 a, b;
                        codes_to_half(w[j], a, b);
                        *reinterpret_cast<uint4*>(tile + to_a + j * kPassRows * 128) = flip ? b : a;
                        *reinterpret_cast<uint4*>(tile + to_b + j * kPassRows * 128) = flip ? a : b;
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[ring]);
                    if (++ring == 3) { ring = 0; ring_phase ^= 1; }
                }
                if (!ok) break;
            }
        }
    } else {
        regs_dec<kIssueRegs>();
    }
    if (warp == 12) {
        // ------------------------------------------------------------------ MMA issue
        constexpr uint32_t idesc_qk = umma_idesc_half(128, false);
        constexpr uint32_t idesc_pv = umma_idesc_half(kDim, true);
        const uint32_t q_addr = smem_u32(smem + L::kQOffset), ring_addr = smem_u32(smem + L::kRingOffset);
        int n_piece = 0;
        uint32_t n_mine = 0;                                  // bit x: parity of the scores asked for of sub-tile x
        int ring_k = 0, ring_v = 1;                           // places of the next K and the next V tile, in turn in the ring
        uint32_t phase_k = 0, phase_v = 0;
        auto advance = [](int& at, uint32_t& phase) {
            at += 2;
            if (at >= 3) { at -= 3; phase ^= 1; }
        };
        for (int u = begin; u < end && ok; ++n_piece) {
            const AttnPiece s = attn_piece<kManyRows, kManyTokens>(p, prefix, u, end);
            u += max(1, s.tile1 - s.tile0);
            const SubTile sub0 = sub_tile(p, s, s.row0, s.row0 + 128), sub1 = sub_tile(p, s, s.row0 + 128, s.row0 + 256);
            ok = attn_wait(q_full, n_piece & 1, abort_flag, p.status, DEV_TIMEOUT_SMEM_FULL);
            if (!ok) break;
            uint32_t started = 0, pending = 0;                // bit x: sub-tile x has had a P V; its last scores have none yet
            for (int t = s.tile0; t <= s.tile1 && ok; ++t) {
                const bool more = t < s.tile1, behind = t > s.tile0;
                const uint32_t k_tile = ring_addr + ring_k * L::kOperandBytes, v_tile = ring_addr + ring_v * L::kOperandBytes;
                const uint32_t active = more ? (sub0.active(t) ? 1u : 0u) | (sub1.active(t) ? 2u : 0u) : 0u;
                // (the operands are there long before the probabilities)
                if (behind) {
                    ok = attn_wait(&full[ring_v], phase_v, abort_flag, p.status, DEV_TIMEOUT_SMEM_FULL);
                    if (!ok) break;
                }
                if (more) {
                    ok = attn_wait(&full[ring_k], phase_k, abort_flag, p.status, DEV_TIMEOUT_SMEM_FULL);
                    if (!ok) break;
                }
                const bool last = t == s.tile1 - 1 || s.tile0 == s.tile1;
#pragma unroll 1
                for (int x = 0; x < 2; ++x) {
                    const uint32_t ts = tmem + x * 128, to = tmem + 256 + x * kDim;
                    const bool pv = pending >> x & 1, qk = active >> x & 1;
                    if (pv) {
                        ok = attn_wait(&p_full[x], ((n_mine >> x) & 1) ^ 1, abort_flag, p.status, DEV_TIMEOUT_TMEM_EMPTY);
                        if (!ok) break;
                    }
                    tcgen05_fence_after();
                    if (elect_one()) {
                        if (pv) {
                            const uint64_t b = umma_desc_sw128_mn(v_tile, 16384);
#pragma unroll
                            for (int k = 0; k < 8; ++k)        // 16 tokens a step: 2048 bytes of V, 8 columns of P
                                umma_f16_ts(to, ts + 8 * k, b + 128 * k, idesc_pv, k > 0 ? 1u : started >> x & 1);
                            umma_commit(&pv_done[x]);
                        }
                        if (qk) {
                            const uint64_t a = umma_desc_sw128(q_addr + x * L::kOperandBytes);
                            const uint64_t b = umma_desc_sw128(k_tile);
#pragma unroll
                            for (int k = 0; k < kDim / 16; ++k) {   // 16 dims a step: 32 bytes, 64 dims a half
                                const uint64_t at = (uint64_t)((k >> 2) * (16384 >> 4) + (k & 3) * 2);
                                umma_f16_ss(ts, a + at, b + at, idesc_qk, k > 0 ? 1u : 0u);
                            }
                            umma_commit(&s_full[x]);
                        }
                        if (x == 1) {
                            if (behind) umma_commit(&free_[ring_v]);
                            if (more) umma_commit(&free_[ring_k]);
                            if (last) umma_commit(q_free);
                        }
                    }
                    __syncwarp();
                    if (pv) {
                        started |= 1u << x;
                        pending &= ~(1u << x);
                    }
                    if (qk) {
                        pending |= 1u << x;
                        n_mine ^= 1u << x;
                    }
                }
                if (!ok) break;
                if (behind) advance(ring_v, phase_v);
                if (more) advance(ring_k, phase_k);
            }
        }
    }
    if (warp == 13) {
        // ------------------------------------------------------------------ pages, scales
        const int bs = cache.block_size;
        const int box_rows = min(bs, 64);
        const uint32_t box_bytes = (uint32_t)box_rows * kDim;
        const int group = lane & 7;                           // of 16 tokens of a tile
        const bool leads = lane < 8 && group * 16 % box_rows == 0;         // this lane's group starts a box
        int n_tile = 0;
        for (int u = begin; u < end && ok;) {
            const AttnPiece s = attn_piece<kManyRows, kManyTokens>(p, prefix, u, end);
            u += max(1, s.tile1 - s.tile0);
            const int* table = p.table + (long long)s.r * p.table_stride;
            // lanes 0..7 hold the blocks of a tile's groups, -1 for one that has none or that nobody sees (read two tiles
            // ahead, looked at one tile later: nothing waits for the table)
            auto wanted = [&](int t) -> bool {
                const int tok = t * kManyTokens + group * 16;
                return t < s.tile1 && tok < s.hi && tok + 16 > s.lo;
            };
            // (a box is fetched when any of its tokens is seen: its first group then looks its block up too)
            auto looked_up = [&](int t) -> bool {
                const int tok = t * kManyTokens + group * 16;
                return t < s.tile1 && (wanted(t) || (leads && tok < s.hi && tok + box_rows > s.lo));
            };
            auto read_block = [&](int t) -> int {
                return looked_up(t) ? table[(t * kManyTokens + group * 16) >> p.block_shift] : -1;
            };
            auto check_block = [&](int t, int block) -> int {
                if (block >= 0 && block < p.num_blocks) return block;
                if (wanted(t)) atomicCAS(p.status, 0, DEV_BAD_CACHE_BLOCK);
                return -1;
            };
            auto scale_of = [&](const float* scales, int block) -> float {
                return block >= 0 ? scales[(long long)block * p.scale_stride + s.head] : 0.0f;
            };
            int blk = check_block(s.tile0, read_block(s.tile0)), raw_block = read_block(s.tile0 + 1);
            float ks = scale_of(p.k_scale, blk), vs = scale_of(p.v_scale, blk);
            for (int t = s.tile0; t < s.tile1; ++t, ++n_tile) {
                const bool seen = blk >= 0 && wanted(t);
                const uint32_t there = __ballot_sync(0xffffffffu, lane < 8 && seen);
                const bool load = leads && blk >= 0;
                const uint32_t loads = __ballot_sync(0xffffffffu, load);
                const int tok = t * kManyTokens + group * 16;
#pragma unroll 1
                for (int which = 0; which < 2; ++which) {
                    ok = attn_wait(&raw_free[which], (n_tile & 1) ^ 1, abort_flag, p.status, DEV_TIMEOUT_SMEM_EMPTY);
                    if (!ok) break;
                    if (which == 0) {
                        if (lane < 8) {
                            const float lv = fmaxf(lg2(vs), kMinLogScale);
                            // (the scores' factor is not negative: the sign of `scale` went into the queries)
                            meta[(n_tile % kManyMeta) * 8 + lane] =
                                make_float4(ks * fabsf(p.scale_log2), seen ? lv : -INFINITY, ex2_subnormal(-lv), __uint_as_float(there));
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&meta_full[n_tile % kManyMeta]);
                    }
                    if (lane == 0) mbar_arrive_expect_tx(&raw_full[which], (uint32_t)__popc(loads) * box_bytes);
                    __syncwarp();
                    if (load)
                        tma_load_page(smem_u32(smem + L::kRawOffset + which * L::kRawBytes) + (uint32_t)group * 16u * kDim,
                                      which ? &map_v : &map_k, smem_u32(&raw_full[which]), tok & (bs - 1), s.head, blk);
                    __syncwarp();
                }
                if (!ok) break;
                blk = check_block(t + 1, raw_block);
                raw_block = read_block(t + 2);
                ks = scale_of(p.k_scale, blk);
                vs = scale_of(p.v_scale, blk);
            }
        }
    }
    grid_launch_dependents();
    __syncthreads();
    if (*abort_flag != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(2000);       // MMAs in flight finish before their memory goes
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 12) {
        __syncwarp();
        tcgen05_fence_after();
        tmem_dealloc<1>(tmem, 512);
    }
}

}  // namespace blaze
