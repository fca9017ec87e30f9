// Attention over the paged 8-bit cache.
//
//   t_j = (q . k8_j) * c_b + L_b      c_b = scale * log2(e) * k_scale_b,  L_b = log2(v_scale_b)
//   m = max t_j - 15,  p_j = 2^(t_j - m),  O = sum p_j v8_j,  l = sum p_j / v_scale_b
//   out = O / l,  lse = (m + log2 l) * ln 2
//
// for the codes k8, v8 of block b's tokens: with the V scale in the exponent neither K nor V is ever multiplied by its
// scale, the codes enter the matrix products as they are (E4M3 is a subset of half), and what is rounded to half is
// p_j relative to the largest p_j * v_scale of its row.  Rounding it is a choice: the codes' own type is the one that the
// products take, and holding p in two halves would double the products with V.  Against 64 bits it costs nothing that bf16
// outputs show (1.4e-3 with p in half as with p in float32), half outputs go from 1.9e-4 to 2.0e-4.
//
// The few-rows kernel (decode steps and short runs of tokens) is bound by the bytes of the cache.  A block has one
// warp that fetches tiles of 64 tokens into a ring in shared memory by TMA (one box per page and operand, 128-byte
// swizzle: 64-byte for 64-wide heads) and four warps that each take 16 of a tile's tokens through both products with
// m16n8k16 instructions, with a running maximum, sum and output of their own, joined once per piece.  Both products are
// computed transposed, S^T = K Q^T and O^T = V^T P^T: the 16 rows of the instruction are tokens or dims, of which there
// are many, its 8 columns the query rows, of which there are few; the probabilities change sides by an 8x8 matrix
// transposition in registers.  The order of the k index of a product is free, so a lane reads 16 consecutive code bytes
// and converts them in registers; the swizzle makes these reads free of bank conflicts for both operands.
// Four contexts of 90k to 131k tokens, 64 query and 8 kv heads of 128: 143 us, 6.2 TB/s (141 without the products); 64
// requests of 200 to 8192 tokens: 118 us, 5.1 TB/s (114 without).  The instance for 9 to 16 rows of 128 spills 96 to 104 bytes at
// its 168 registers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cmath>

#include "cache.h"
#include "cache_attention_many.cuh"
#include "cache_schedule.cuh"
#include "cann_ops_tensor_types.h"
#include "launch.h"
#include "ptx.cuh"

namespace blaze {

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kFewRows = 16;          // packed rows of a row tile, at most: 8 for each n8 tile of the products
constexpr int kFewTokens = 64;        // tokens of a tile
constexpr int kFewWarps = 4;          // computing warps, 16 tokens of a tile each
constexpr int kFewThreads = 32 * (kFewWarps + 1);
constexpr int kFewStages = 4;
// Tiles of a block's chunk, at least.  1, 2 and 4 of them: one token on 1000 tokens 11.0, 9.2 and 9.0 us, on 300 tokens 7.9,
// 10.2 and 10.7; a prompt of 512 tokens (many rows) 39.5, 39.6 and 50.
constexpr int kFewMinChunk = 2;
constexpr int kManyMinChunk = 2;
// Requests of more packed rows go to the many-rows kernel: this one reads the cache once per 16 rows, that one once per 256 at
// the price of 256 rows' products.  Measured, few-rows / many-rows kernel in us, 2 kv heads, 16 requests of 2k tokens, 4 of 30k
// and 32 of 8k: heads of 128, 24 rows 30 / 26, 48 / 57, 84 / 92; 32 rows 32 / 26, 49 / 58, 87 / 94; 40 rows 34 / 27, 61 / 59,
// 113 / 94; 72 rows 42 / 28, 84 / 64, 166 / 97.  Heads of 64, 32 rows 22 / 22, 35 / 46, 55 / 72; 48 rows 25 / 22, 41 / 47, 71 / 74;
// 64 rows 27 / 22, 47 / 48, 87 / 75.  So up to 32 rows of 128 each is ahead by 10 to 20 % somewhere, and for heads of 64 this
// one would be ahead up to 48 rows on long contexts.
constexpr int kFewLimit = kFewRows;
// Small calls stay with the few-rows kernel whatever their rows: up to so many tiles of 64 tokens per block, counting 16 rows
// a row tile and every request as long as the longest.  Measured, few-rows / many-rows kernel: 0.2 tiles (420 rows on 105
// tokens) 12 / 21 us; 3.9 (17 requests of up to 374 rows on up to 291 tokens) 27 / 53; 11.6 (8 of up to 160 rows on up to 340)
// 41 / 33; 31 (2048 rows on 512) 96 / 40.
constexpr double kFewSmall = 6.0;

// Probabilities are kept up to 2^15 (the running maximum less 15), so that in half the values down to 2^-29 of a row's
// largest have all their 11 bits and nothing above 2^-40 of it vanishes, however long the row.
constexpr float kProbShift = 15.0f;

template <int kDim>
struct FewSmem {
    static constexpr int kBlocks = kDim == 64 ? 3 : 2;               // resident blocks of an SM
    static constexpr int kTileBytes = kFewTokens * kDim;             // of K, and of V
    static constexpr int kStageBytes = 2 * kTileBytes;
    static constexpr int kPitch = kDim + 4;                          // floats of a row of a warp's output
    static constexpr int kJoinOffset = kFewStages * kStageBytes;
    static constexpr int kMlOffset = kJoinOffset + kFewWarps * kFewRows * kPitch * 4;
    static constexpr int kMetaOffset = kMlOffset + kFewWarps * kFewRows * 2 * 4;    // float4 per stage and warp
    static constexpr int kBarOffset = kMetaOffset + kFewStages * kFewWarps * 16;
    static constexpr int kMiscOffset = kBarOffset + (2 * kFewStages + 2) * 8;
    static constexpr int kPrefixOffset = kMiscOffset + 64;
    static int bytes(int requests) { return 1024 + kPrefixOffset + (requests + 1) * 4; }
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 0xFF in every byte that is an E4M3 NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// Transpose of an 8x8 matrix of halves held two to a lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int kDim, bool kBf16, int kTiles>
__global__ void __launch_bounds__(kFewThreads, FewSmem<kDim>::kBlocks)
cache_attention_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const CacheAttentionParams p) {
    using L = FewSmem<kDim>;
    constexpr int kRows = 8 * kTiles;          // query rows of a row tile, in kTiles n8 tiles
    constexpr int kSteps = kDim / 16;          // k16 steps of K Q^T
    constexpr int kBands = kDim / 16;          // m16 tiles of V^T P^T
    constexpr int kLaneDims = kDim / 8;        // consecutive dims of O of a lane
    extern __shared__ uint8_t few_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(few_smem_raw) + 1023) & ~uintptr_t(1023));
    float* join = reinterpret_cast<float*>(smem + L::kJoinOffset);
    float* ml = reinterpret_cast<float*>(smem + L::kMlOffset);
    float4* meta = reinterpret_cast<float4*>(smem + L::kMetaOffset);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOffset);
    uint64_t* empty = full + kFewStages;
    uint64_t* joined = empty + kFewStages;         // the computing warps meet here
    int* misc = reinterpret_cast<int*>(smem + L::kMiscOffset);
    volatile int* abort_flag = misc + 8;
    int* prefix = reinterpret_cast<int*>(smem + L::kPrefixOffset);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kFewStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kFewWarps);
        }
        mbar_init(joined, kFewWarps);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
    }
    grid_dependency_wait();
    attn_prefix<kRows, kFewTokens>(p, prefix, misc);
    const int total = prefix[p.requests];
    const int chunk = attn_chunk(p, total, gridDim.x);
    const long long begin64 = (long long)blockIdx.x * chunk;
    const int begin = (int)min(begin64, (long long)total);
    const int end = (int)min(begin64 + chunk, (long long)total);
    if (threadIdx.x == 0) p.cuts[blockIdx.x].first = -1;          // until this thread knows better

    if (warp == kFewWarps) {
        // ------------------------------------------------------------------ fetching warp
        const int bs = 1 << p.block_shift;
        const int box_rows = min(bs, kFewTokens);
        const uint32_t box_bytes = (uint32_t)box_rows * kDim;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int u = begin; u < end && ok;) {
            const AttnPiece s = attn_piece<kRows, kFewTokens>(p, prefix, u, end);
            u += max(1, s.tile1 - s.tile0);
            const int* table = p.table + (long long)s.r * p.table_stride;
            // Lane i holds page `base + i` of the request: block number and scales, fetched 32 pages at a time and one
            // batch ahead of their use.  A batch starts at the page of a tile's first token, so no tile crosses one.
            auto fetch = [&](int base, int& block, float& ks, float& vs) {
                const int page = base + lane;
                const bool in = page < p.max_blocks && ((page + 1) << p.block_shift) > s.lo && (page << p.block_shift) < s.hi;
                block = in ? table[page] : -1;
                if (in && (block < 0 || block >= p.num_blocks)) {
                    atomicCAS(p.status, 0, DEV_BAD_CACHE_BLOCK);
                    block = -1;
                }
                ks = vs = 0.0f;
                if (block >= 0) {
                    ks = p.k_scale[(long long)block * p.scale_stride + s.head];
                    vs = p.v_scale[(long long)block * p.scale_stride + s.head];
                }
            };
            int base = (s.tile0 * kFewTokens) >> p.block_shift;
            int blk, blk2;
            float ks, vs, ks2, vs2;
            fetch(base, blk, ks, vs);
            fetch(base + 32, blk2, ks2, vs2);
            for (int t = s.tile0; t < s.tile1; ++t) {
                const int page0 = (t * kFewTokens) >> p.block_shift;
                if (page0 >= base + 32) {
                    base += 32;
                    blk = blk2; ks = ks2; vs = vs2;
                    fetch(base + 32, blk2, ks2, vs2);
                }
                // lanes 0..3: the tile's groups of 16 tokens
                const int tok = t * kFewTokens + (lane & 3) * 16;
                const int src = (tok >> p.block_shift) - base;
                const int block = __shfl_sync(0xffffffffu, blk, src);
                const float k_s = __shfl_sync(0xffffffffu, ks, src), v_s = __shfl_sync(0xffffffffu, vs, src);
                ok = mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.status, DEV_TIMEOUT_SMEM_EMPTY);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                // a box (a page, or 64 tokens of one) is loaded when any of its tokens is seen and its block exists
                const bool leader = lane < 4 && (lane * 16) % box_rows == 0;
                const bool load = leader && block >= 0 && tok < s.hi && tok + box_rows > s.lo;
                const uint32_t loads = __ballot_sync(0xffffffffu, load);
                if (lane < 4) {
                    const bool seen = block >= 0 && tok < s.hi && tok + 16 > s.lo;
                    const float lv = fmaxf(lg2(v_s), kMinLogScale);
                    meta[stage * kFewWarps + lane] =
                        make_float4(k_s * p.scale_log2, seen ? lv : -INFINITY, ex2_subnormal(-lv), 0.0f);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(&full[stage], (uint32_t)__popc(loads) * 2u * box_bytes);
                __syncwarp();
                if (load) {
                    const uint32_t dst = smem_u32(smem + stage * L::kStageBytes) + (uint32_t)lane * 16u * kDim;
                    const uint32_t bar = smem_u32(&full[stage]);
                    const int row = tok & (bs - 1);
                    tma_load_page(dst, &map_k, bar, row, s.head, block);
                    tma_load_page(dst + L::kTileBytes, &map_v, bar, row, s.head, block);
                }
                __syncwarp();
                if (++stage == kFewStages) { stage = 0; phase ^= 1; }
            }
        }
        grid_launch_dependents();
    } else {
        // ------------------------------------------------------------------ computing warps
        // g: a token (and the one 8 behind it) or a band of dims, and the query row whose B operand the lane has;
        // rows 2c, 2c + 1 of each n8 tile are the ones whose scores, statistics and output it has
        const int g = lane >> 2, c = lane & 3;
        int stage = 0;
        uint32_t phase = 0, meeting = 0;
        bool ok = true;
        // A meeting of the computing warps, bounded like every wait: a warp that has given up elsewhere does not come.
        auto meet = [&]() -> bool {
            __syncwarp();
            if (lane == 0) mbar_arrive(joined);
            const bool there = mbar_wait(joined, meeting, abort_flag, p.status, DEV_TIMEOUT_SMEM_EMPTY);
            meeting ^= 1;
            return __all_sync(0xffffffffu, there);
        };
        for (int u = begin; u < end && ok;) {
            const AttnPiece s = attn_piece<kRows, kFewTokens>(p, prefix, u, end);
            const int u_next = u + max(1, s.tile1 - s.tile0);
            const int off = s.req.kv - s.req.qlen;
            auto see = [&](int row, int& lo, int& hi) {            // tokens that a row of the tile sees
                const int i = row / p.group;
                hi = row < s.rows ? (p.causal ? min(s.req.kv, off + i + 1) : s.req.kv) : 0;
                lo = p.window > 0 ? max(0, off + i - p.window + 1) : 0;
            };
            // ---- queries: the B operand of row g of each tile, as half
            uint32_t qf[kTiles][kSteps][2];
            float factor[kTiles][2];                   // of the scores of rows 2c, 2c + 1
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                const int row = s.row0 + 8 * n + g;
                const bool there = row < s.rows;
                const int i = there ? row / p.group : 0;
                const int head = s.head * p.group + (there ? row - i * p.group : 0);
                const uint16_t* src = static_cast<const uint16_t*>(p.q) + (long long)(s.req.q0 + i) * p.q_token_stride +
                                      (long long)head * p.q_head_stride;
                uint4 w[kSteps / 2];                   // 16 dims (two loads) for every four steps
#pragma unroll
                for (int k = 0; k < kSteps / 2; ++k) {
                    const int dim = kDim == 128 ? (2 * c + (k >> 1)) * 16 + (k & 1) * 8 : c * 16 + k * 8;
                    w[k] = there ? *reinterpret_cast<const uint4*>(src + dim) : make_uint4(0, 0, 0, 0);
                }
                float mul = 1.0f, back = 1.0f;
                if constexpr (kBf16) {
                    float amax = 0.0f;
#pragma unroll
                    for (int k = 0; k < kSteps / 2; ++k) {
                        const uint32_t* x = &w[k].x;
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const uint32_t a = x[h] & 0x7FFFu, b = (x[h] >> 16) & 0x7FFFu;
                            amax = fmaxf(amax, __uint_as_float((a < 0x7F80u ? a : 0u) << 16));
                            amax = fmaxf(amax, __uint_as_float((b < 0x7F80u ? b : 0u) << 16));
                        }
                    }
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                    const int shift = query_shift(amax);
                    mul = pow2i(shift);
                    back = pow2i(-shift);
                }
                // row r's factor is with the lanes of g = r
                factor[n][0] = __shfl_sync(0xffffffffu, back, 8 * c);
                factor[n][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
#pragma unroll
                for (int k = 0; k < kSteps / 2; ++k) {
                    const uint32_t* x = &w[k].x;
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        uint32_t v = x[h];
                        if constexpr (kBf16)
                            v = pack_f16(__uint_as_float(v << 16) * mul, __uint_as_float(v & 0xFFFF0000u) * mul);
                        qf[n][2 * k + (h >> 1)][h & 1] = v;        // words 0, 1: step 2k; words 2, 3: step 2k + 1
                    }
                }
            }
            // every row of the tile sees the tokens [all_lo, all_hi)
            const int i_first = s.row0 / p.group, i_last = (min(s.rows, s.row0 + kRows) - 1) / p.group;
            const int all_hi = p.causal ? min(s.req.kv, off + i_first + 1) : s.req.kv;
            const int all_lo = p.window > 0 ? max(0, off + i_last - p.window + 1) : 0;

            float o[kTiles][kBands][4];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                for (int j = 0; j < kBands; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
            }
            float m[kTiles][2], l[kTiles][2];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                m[n][0] = m[n][1] = -INFINITY;
                l[n][0] = l[n][1] = 0.0f;
            }

            for (int t = s.tile0; t < s.tile1; ++t) {
                ok = mbar_wait(&full[stage], phase, abort_flag, p.status, DEV_TIMEOUT_SMEM_FULL);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const float4 mt = meta[stage * kFewWarps + warp];
                const int tok0 = t * kFewTokens + warp * 16;
                const uint8_t* kt = smem + stage * L::kStageBytes;
                const uint8_t* vt = kt + L::kTileBytes;
                if (mt.y != -INFINITY) {               // same for the whole warp
                    // ---- scores of tokens g, g + 8 and rows 2c, 2c + 1, 16 codes of a token at a time
                    float sc[kTiles][4];
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
#pragma unroll
                    for (int i = 0; i < kDim / 64; ++i) {
                        uint4 w[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int row = warp * 16 + h * 8 + g;
                            w[h] = kDim == 128
                                ? *reinterpret_cast<const uint4*>(kt + row * 128 + (((2 * c + i) ^ (row & 7)) << 4))
                                : *reinterpret_cast<const uint4*>(kt + row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t w0 = (&w[0].x)[j], w1 = (&w[1].x)[j];
                            const uint32_t a[4] = {codes_lo(w0), codes_lo(w1), codes_hi(w0), codes_hi(w1)};
#pragma unroll
                            for (int n = 0; n < kTiles; ++n) mma_f16(sc[n], a, qf[n][4 * i + j][0], qf[n][4 * i + j][1]);
                        }
                    }
                    // ---- V codes of the tokens 2c, 2c + 1, 2c + 8, 2c + 9, dims [g * kDim / 8, (g + 1) * kDim / 8)
                    uint32_t wv[4][kDim / 32];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int row = warp * 16 + 2 * c + (k & 1) + (k >> 1) * 8;
                        if constexpr (kDim == 128) {
                            const uint4 w = *reinterpret_cast<const uint4*>(vt + row * 128 + ((g ^ (row & 7)) << 4));
                            wv[k][0] = w.x; wv[k][1] = w.y; wv[k][2] = w.z; wv[k][3] = w.w;
                        } else {
                            const uint2 w = *reinterpret_cast<const uint2*>(vt + row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + (g & 1) * 8);
                            wv[k][0] = w.x; wv[k][1] = w.y;
                        }
                    }
                    // band j is dims 2j (instruction rows 0..7) and 2j + 1 (rows 8..15) of every lane's dims
                    auto band = [&](const uint32_t (&w)[4][kDim / 32], int j, uint32_t (&a)[4]) {
                        const int i = j >> 1, sel = (j & 1) ? 0x7362 : 0x5140;
                        const uint32_t x = __byte_perm(w[0][i], w[1][i], sel), y = __byte_perm(w[2][i], w[3][i], sel);
                        a[0] = codes_lo(x); a[1] = codes_hi(x); a[2] = codes_lo(y); a[3] = codes_hi(y);
                    };
                    // ---- softmax
                    const bool masked = tok0 < all_lo || tok0 + 16 > all_hi;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        const float f0 = factor[n][0] * mt.x, f1 = factor[n][1] * mt.x;
                        sc[n][0] = fmaf(sc[n][0], f0, mt.y);
                        sc[n][1] = fmaf(sc[n][1], f1, mt.y);
                        sc[n][2] = fmaf(sc[n][2], f0, mt.y);
                        sc[n][3] = fmaf(sc[n][3], f1, mt.y);
                    }
                    if (masked) {
#pragma unroll
                        for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                int lo, hi;
                                see(s.row0 + 8 * n + 2 * c + e, lo, hi);
                                if (tok0 + g < lo || tok0 + g >= hi) sc[n][e] = -INFINITY;
                                if (tok0 + g + 8 < lo || tok0 + g + 8 >= hi) sc[n][2 + e] = -INFINITY;
                            }
                        }
                        // codes of tokens outside the item do not count; NaN codes of tokens that some rows see and
                        // others do not are taken out of the product, and the rows that see them are given their NaN
                        // by a product of ones: is-NaN x seen
                        bool any = false;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int tok = tok0 + 2 * c + (k & 1) + (k >> 1) * 8;
#pragma unroll
                            for (int i = 0; i < kDim / 32; ++i) {
                                if (tok < s.lo || tok >= s.hi) wv[k][i] = 0;
                                any |= nan_bytes(wv[k][i]) != 0;
                            }
                        }
                        if (__any_sync(0xffffffffu, any)) {
                            uint32_t wn[4][kDim / 32];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
#pragma unroll
                                for (int i = 0; i < kDim / 32; ++i) {
                                    const uint32_t nb = nan_bytes(wv[k][i]);
                                    wn[k][i] = nb & 0x38383838u;      // E4M3 one
                                    wv[k][i] &= ~nb;
                                }
                            }
#pragma unroll
                            for (int n = 0; n < kTiles; ++n) {
                                int lo, hi;
                                see(s.row0 + 8 * n + g, lo, hi);
                                uint32_t ones[2];
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    const int tok = tok0 + 2 * c + 8 * k;
                                    ones[k] = (tok >= lo && tok < hi ? 0x3C00u : 0u) | (tok + 1 >= lo && tok + 1 < hi ? 0x3C000000u : 0u);
                                }
#pragma unroll
                                for (int j = 0; j < kBands; ++j) {
                                    uint32_t a[4];
                                    band(wn, j, a);
                                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                    mma_f16(d, a, ones[0], ones[1]);
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        if (d[e] > 0.0f) o[n][j][e] = NAN;
                                }
                            }
                        }
                    }
                    uint32_t pf[kTiles][2];
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        float mx[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            mx[e] = fmaxf(sc[n][e], sc[n][2 + e]);
                            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 4));
                            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 8));
                            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 16));
                            mx[e] = fmaxf(m[n][e], mx[e] - kProbShift);
                        }
                        if (__any_sync(0xffffffffu, mx[0] > m[n][0] || mx[1] > m[n][1])) {
                            float al[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                al[e] = m[n][e] == mx[e] ? 1.0f : (m[n][e] == -INFINITY ? 0.0f : ex2(m[n][e] - mx[e]));
                                m[n][e] = mx[e];
                                l[n][e] *= al[e];
                            }
#pragma unroll
                            for (int j = 0; j < kBands; ++j) {
                                o[n][j][0] *= al[0]; o[n][j][1] *= al[1];
                                o[n][j][2] *= al[0]; o[n][j][3] *= al[1];
                            }
                        }
                        const float ms0 = m[n][0] == -INFINITY ? 0.0f : m[n][0], ms1 = m[n][1] == -INFINITY ? 0.0f : m[n][1];
                        const float p0 = ex2(sc[n][0] - ms0), p1 = ex2(sc[n][1] - ms1);
                        const float p2 = ex2(sc[n][2] - ms0), p3 = ex2(sc[n][3] - ms1);
                        l[n][0] = fmaf(p0 + p2, mt.z, l[n][0]);
                        l[n][1] = fmaf(p1 + p3, mt.z, l[n][1]);
                        pf[n][0] = transpose8x8(pack_f16(p0, p1));
                        pf[n][1] = transpose8x8(pack_f16(p2, p3));
                    }
                    // ---- V^T P^T
#pragma unroll
                    for (int j = 0; j < kBands; ++j) {
                        uint32_t a[4];
                        band(wv, j, a);
#pragma unroll
                        for (int n = 0; n < kTiles; ++n) mma_f16(o[n][j], a, pf[n][0], pf[n][1]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[stage]);
                if (++stage == kFewStages) { stage = 0; phase ^= 1; }
            }
            if (!ok) break;
            // ---- join the four warps: this lane has rows 2c, 2c + 1, dims [g * kLaneDims, (g + 1) * kLaneDims)
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float sum = l[n][e];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    const int row = 8 * n + 2 * c + e;
                    if (g == 0) *reinterpret_cast<float2*>(ml + (warp * kFewRows + row) * 2) = make_float2(m[n][e], sum);
                    // (in an order that keeps lanes of different g on different banks)
                    float* dst = join + (warp * kFewRows + row) * L::kPitch + g * kLaneDims;
#pragma unroll
                    for (int k = 0; k < kLaneDims; k += 4)
                        *reinterpret_cast<float4*>(dst + k) = make_float4(o[n][k / 2][e], o[n][k / 2][2 + e], o[n][k / 2 + 1][e], o[n][k / 2 + 1][2 + e]);
                }
            }
            ok = meet();
            if (!ok) break;
            {
                constexpr int kPer = kDim * kRows / (32 * kFewWarps);       // dims of this thread
                constexpr int kPerRow = kDim / kPer;                        // threads of a row
                const int tid = threadIdx.x;           // the computing warps are the block's first
                const int row = tid / kPerRow, d0 = (tid % kPerRow) * kPer;
                float mm = -INFINITY, ll = 0.0f, acc[kPer];
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w) mm = fmaxf(mm, ml[(w * kFewRows + row) * 2]);
#pragma unroll
                for (int k = 0; k < kPer; ++k) acc[k] = 0.0f;
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w) {
                    const float2 v = *reinterpret_cast<const float2*>(ml + (w * kFewRows + row) * 2);
                    const float wt = v.x == -INFINITY ? 0.0f : ex2(v.x - mm);
                    ll += wt * v.y;                    // (0 * NaN for a warp all of whose scores are NaN: so is the row)
                    if (wt == 0.0f) continue;
                    const float* src = join + (w * kFewRows + row) * L::kPitch + d0;
#pragma unroll
                    for (int k = 0; k < kPer; k += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(src + k);
                        acc[k] = fmaf(wt, x.x, acc[k]);
                        acc[k + 1] = fmaf(wt, x.y, acc[k + 1]);
                        acc[k + 2] = fmaf(wt, x.z, acc[k + 2]);
                        acc[k + 3] = fmaf(wt, x.w, acc[k + 3]);
                    }
                }
                const int prow = s.row0 + row;
                if (prow < s.rows) {
                    const bool whole = s.item0 >= begin && s.item1 <= end;
                    if (whole) {
                        const int i = prow / p.group;
                        const int head = s.head * p.group + (prow - i * p.group);
                        const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
                        uint16_t* dst = static_cast<uint16_t*>(p.out) + (long long)(s.req.q0 + i) * p.out_token_stride +
                                        (long long)head * p.out_head_stride + d0;
#pragma unroll
                        for (int k = 0; k < kPer; k += 4)
                            *reinterpret_cast<uint2*>(dst + k) = make_uint2(pack_out<kBf16>(acc[k] * inv, acc[k + 1] * inv),
                                                                            pack_out<kBf16>(acc[k + 2] * inv, acc[k + 3] * inv));
                        if (p.lse && tid % kPerRow == 0)
                            p.lse[(long long)(s.req.q0 + i) * p.heads + head] =
                                ll != 0.0f ? (mm + lg2(ll)) * 0.6931471805599453f : -INFINITY;
                    } else {
                        const long long slot = (long long)blockIdx.x * 2 + (u == begin ? 0 : 1);
                        float* dst = p.part_out + (slot * kRows + row) * kDim + d0;
#pragma unroll
                        for (int k = 0; k < kPer; k += 4)
                            *reinterpret_cast<float4*>(dst + k) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
                        if (tid % kPerRow == 0)
                            *reinterpret_cast<float2*>(p.part_ml + (slot * kRows + row) * 2) = make_float2(mm, ll);
                    }
                }
            }
            if (threadIdx.x == 0 && u_next >= end) attn_write_cut(p, s, blockIdx.x, chunk, end);
            ok = meet();
            u = u_next;
        }
        grid_launch_dependents();
    }
    // (a block whose wait ran out leaves with copies in flight: give them time to land before its memory is reused)
    __syncthreads();
    if (*abort_flag != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(2000);
    }
}

// Joins the pieces of the items that are cut by a chunk's border: out = sum_b w_b O_b / sum_b w_b l_b with w_b = 2^(m_b -
// max m), in the order of the blocks.  Block `which` takes the item that the end of that block's chunk cuts, unless the
// item was cut before; a large row tile is shared by kRows / 16 blocks, whose warps take rows.  Bound by latency: the
// statistics of 32 pieces are read at once by a warp's lanes, then four pieces of output are in flight.
template <int kRows, int kDim, bool kBf16>
__global__ void __launch_bounds__(256) cache_attention_join_kernel(const CacheAttentionParams p) {
    constexpr int kGroups = kRows > 16 ? kRows / 16 : 1;
    constexpr int kPer = kDim / 32;
    grid_launch_dependents();
    grid_dependency_wait();
    const int which = blockIdx.x / kGroups, group = blockIdx.x % kGroups;
    const AttnCut s = p.cuts[which];
    if (s.first != which) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = min(min((group + 1) * 16, kRows), s.rows - s.row0);
    const int pieces = s.last - s.first + 1;
    // slot 0 of a block is the piece at the start of its chunk, slot 1 one that starts inside it
    auto slot_of = [&](int b) -> long long { return (long long)(s.first + b) * 2 + (b == 0 ? s.inside : 0); };
    for (int row = group * 16 + warp; row < rows; row += 8) {
        float mm = -INFINITY, ll = 0.0f, acc[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) acc[k] = 0.0f;
#pragma unroll 1
        for (int b0 = 0; b0 < pieces; b0 += 32) {
            float2 v = make_float2(-INFINITY, 0.0f);
            if (b0 + lane < pieces) v = *reinterpret_cast<const float2*>(p.part_ml + (slot_of(b0 + lane) * kRows + row) * 2);
            float m_new = v.x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, o));
            m_new = fmaxf(m_new, mm);
            // (a piece that saw nothing has weight 0, but its sum may be the NaN of a score)
            const float w = v.x == -INFINITY ? 0.0f : ex2(v.x - m_new);
            const float keep = mm == -INFINITY ? 0.0f : ex2(mm - m_new);
            mm = m_new;
            float sum = w * v.y;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            ll = ll * keep + sum;
#pragma unroll
            for (int k = 0; k < kPer; ++k) acc[k] *= keep;
            const int n = min(32, pieces - b0);
#pragma unroll 1
            for (int b = 0; b < n; b += 4) {
                float x[4][kPer];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float* src = p.part_out + (slot_of(b0 + min(b + j, n - 1)) * kRows + row) * kDim + lane * kPer;
#pragma unroll
                    for (int k = 0; k < kPer; ++k) x[j][k] = src[k];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float wj = __shfl_sync(0xffffffffu, w, (b + j) & 31);
                    if (b + j < n && wj != 0.0f) {
#pragma unroll
                        for (int k = 0; k < kPer; ++k) acc[k] = fmaf(wj, x[j][k], acc[k]);
                    }
                }
            }
        }
        const int prow = s.row0 + row;
        const int i = prow / p.group;
        const int head = s.head * p.group + (prow - i * p.group);
        const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + (long long)(s.q0 + i) * p.out_token_stride +
                        (long long)head * p.out_head_stride + lane * kPer;
#pragma unroll
        for (int k = 0; k < kPer; k += 2)
            *reinterpret_cast<uint32_t*>(dst + k) = pack_out<kBf16>(acc[k] * inv, acc[k + 1] * inv);
        if (p.lse && lane == 0)
            p.lse[(long long)(s.q0 + i) * p.heads + head] =
                ll != 0.0f ? (mm + lg2(ll)) * 0.6931471805599453f : -INFINITY;
    }
}

// ---------------------------------------------------------------------------------------------------- launch

// One page, or `box_rows` tokens of one, per box; the coordinates are (dim, token in block, head, block).
static bool make_tmap_pages(CUtensorMap* map, const void* base, const blazeKvCache* c, int box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->block_size, (cuuint64_t)c->kv_heads,
                                (cuuint64_t)c->num_blocks};
    // (the stride of a dimension of one is never used, but has to be a legal one)
    const cuuint64_t token = (cuuint64_t)c->token_stride;
    const cuuint64_t strides[3] = {token, c->kv_heads > 1 ? (cuuint64_t)c->head_stride : token,
                                   c->num_blocks > 1 ? (cuuint64_t)c->block_stride : token};
    const cuuint32_t box[4] = {(cuuint32_t)c->head_dim, (cuuint32_t)box_rows, 1, 1};
    const cuuint32_t elem_strides[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, elem_strides,
              CU_TENSOR_MAP_INTERLEAVE_NONE, c->head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Which kernels a call needs, by the bounds of its requests' rows, and where their partial results lie.
struct AttnPlan {
    bool few, many;
    int few_rows;                                      // packed rows up to which a request is the few-rows kernel's
    int few_grid, many_grid;
    size_t few_ml, few_cuts, many_out, many_ml, many_cuts, total;      // offsets in the workspace (few_out is 0)
};

static int plan_attention(const blazeKvCache* c, const blazeCacheAttentionArgs* a, int sms, AttnPlan* pl) {
    const int st = check_kv_cache(c);
    if (st != ACLTENSOR_STATUS_SUCCESS) return st;
    if (!a || a->struct_size < sizeof(blazeCacheAttentionArgs)) return ACLTENSOR_STATUS_INVALID_VALUE;
    if (a->requests < 0 || a->tokens < 0 || a->heads < 1 || (a->heads % c->kv_heads) || a->max_q < 0 || a->min_q < 0 ||
        a->max_kv < 0 || a->max_blocks < 0 || a->window < 0 || a->sm_limit < 0 || (a->causal != 0 && a->causal != 1) ||
        a->table_stride < a->max_blocks || (int64_t)a->max_kv > (int64_t)a->max_blocks * c->block_size ||
        !std::isfinite(a->scale * kLog2E))            // (scores are taken as powers of two)
        return ACLTENSOR_STATUS_INVALID_VALUE;
    if (a->requests > kAttnMaxRequests || (a->q_type != BLAZE_OUT_BF16 && a->q_type != BLAZE_OUT_F16))
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    const int64_t group = a->heads / c->kv_heads, rows = (int64_t)a->max_q * group;
    if (a->max_kv > (1 << 30) || rows > (1 << 24)) return ACLTENSOR_STATUS_NOT_SUPPORTED;
    // units are counted in 32 bits
    const double heads = (double)a->requests * c->kv_heads;
    if (heads * (double)(a->max_kv / kFewTokens + 2) > 2.0e9 ||
        (rows > kFewLimit && heads * (double)((rows + kManyRows - 1) / kManyRows) * (double)(a->max_kv / kManyTokens + 2) > 2.0e9))
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    if (a->sm_limit > 0 && a->sm_limit < sms) sms = a->sm_limit;
    // (a long prefix over many requests may leave no room for the last block of an SM)
    const int few_bytes = c->head_dim == 128 ? FewSmem<128>::bytes(a->requests) : FewSmem<64>::bytes(a->requests);
    const int few_blocks = c->head_dim == 128 ? FewSmem<128>::kBlocks : FewSmem<64>::kBlocks;
    const int fit = (228 * 1024) / (few_bytes + 1024);
    pl->few_grid = (fit < few_blocks ? fit : few_blocks) * sms;
    pl->many_grid = sms;
    // tiles of 64 tokens per block if the few-rows kernel took everything, at most
    const double few_tiles = c->kv_heads * ((double)a->tokens * group / kFewRows + a->requests) *
                             (a->max_kv / kFewTokens + 1.0) / pl->few_grid;
    const bool small = few_tiles <= kFewSmall;
    pl->many = rows > kFewLimit && !small;
    pl->few = !pl->many || (int64_t)a->min_q * group <= kFewLimit;
    pl->few_rows = small ? 0x7FFFFFFF : kFewLimit;
    size_t at = 0;
    auto room = [&](int grid, int tile_rows, size_t* ml, size_t* cuts) {
        at += round256((size_t)grid * 2 * tile_rows * c->head_dim * 4);
        *ml = at;
        at += round256((size_t)grid * 2 * tile_rows * 2 * 4);
        *cuts = at;
        at += round256((size_t)grid * sizeof(AttnCut));
    };
    pl->few_ml = pl->few_cuts = pl->many_out = pl->many_ml = pl->many_cuts = 0;
    // (room for all the blocks that a call of fewer requests may have: what suffices for larger bounds suffices for smaller)
    if (pl->few) room(few_blocks * sms, kFewRows, &pl->few_ml, &pl->few_cuts);
    pl->many_out = at;
    if (pl->many) room(pl->many_grid, kManyRows, &pl->many_ml, &pl->many_cuts);
    pl->total = at;
    return ACLTENSOR_STATUS_SUCCESS;
}

// What the kernels of a head size and type need before their first launch on a device.  The ones that the call at hand does
// not launch are loaded too, so that a capture may follow any first call; only a call that needs the many-rows kernel
// fails where that one cannot run.
template <int kDim, bool kBf16>
static cudaError_t prepare_attention(bool with_many) {
    enum { kUnknown, kAll, kWithoutMany };
    static int state[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    int& known = state[dev & 63];
    if (known == kUnknown) {
        static_assert(1024 + FewSmem<kDim>::kPrefixOffset + (kAttnMaxRequests + 1) * 4 <= 227 * 1024, "shared memory");
        static_assert(1024 + ManySmem<kDim>::kPrefixOffset + (kAttnMaxRequests + 1) * 4 <= 227 * 1024, "shared memory");
        const cudaFuncAttribute smem = cudaFuncAttributeMaxDynamicSharedMemorySize;
        const int few_bytes = FewSmem<kDim>::bytes(kAttnMaxRequests);
        cudaFuncAttributes attr;
        cudaError_t e = cudaFuncSetAttribute(cache_attention_few_kernel<kDim, kBf16, 1>, smem, few_bytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(cache_attention_few_kernel<kDim, kBf16, 2>, smem, few_bytes);
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, cache_attention_join_kernel<8, kDim, kBf16>);
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, cache_attention_join_kernel<16, kDim, kBf16>);
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, cache_attention_join_kernel<kManyRows, kDim, kBf16>);
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, cache_attention_many_kernel<kDim, kBf16>);
        if (e != cudaSuccess) return e;
        // its warpgroups trade registers: the launch has to have all that they take (the build checks it too)
        const bool many = attr.numRegs >= kManyLaunchRegs;
        if (many)
            e = cudaFuncSetAttribute(cache_attention_many_kernel<kDim, kBf16>, smem, ManySmem<kDim>::bytes(kAttnMaxRequests));
        if (e != cudaSuccess) return e;
        known = many ? kAll : kWithoutMany;
    }
    return with_many && known != kAll ? cudaErrorInvalidConfiguration : cudaSuccess;
}

template <int kDim, bool kBf16, int kTiles>
static cudaError_t launch_few(const CUtensorMap& mk, const CUtensorMap& mv, const CacheAttentionParams& p, int grid,
                              cudaStream_t stream) {
    auto few = cache_attention_few_kernel<kDim, kBf16, kTiles>;
    const cudaError_t e = launch_after_prepass(few, grid, kFewThreads, (size_t)FewSmem<kDim>::bytes(p.requests), stream, mk, mv, p);
    if (e != cudaSuccess || grid < 2) return e;
    return launch_after_prepass(cache_attention_join_kernel<8 * kTiles, kDim, kBf16>, grid - 1, 256, 0, stream, p);
}

template <int kDim, bool kBf16>
static cudaError_t launch_attention(const CUtensorMap& mk, const CUtensorMap& mv, CacheAttentionParams p, const CacheView& cv,
                                    const AttnPlan& pl, uint8_t* ws, cudaStream_t stream) {
    cudaError_t e = prepare_attention<kDim, kBf16>(pl.many);
    if (e != cudaSuccess) return e;
    p.few_rows = pl.few_rows;
    if (pl.few) {
        p.take_few = 1;
        p.take_many = 0;
        p.min_chunk = kFewMinChunk;
        p.part_out = reinterpret_cast<float*>(ws);
        p.part_ml = reinterpret_cast<float*>(ws + pl.few_ml);
        p.cuts = reinterpret_cast<AttnCut*>(ws + pl.few_cuts);
        // a second n8 tile of query rows only where a request may need it
        e = (long long)p.max_q * p.group <= 8 ? launch_few<kDim, kBf16, 1>(mk, mv, p, pl.few_grid, stream)
                                              : launch_few<kDim, kBf16, 2>(mk, mv, p, pl.few_grid, stream);
        if (e != cudaSuccess) return e;
    }
    if (pl.many) {
        p.take_few = pl.few ? 0 : 1;                   // (without the few-rows launch every request is this one's)
        p.take_many = 1;
        p.min_chunk = kManyMinChunk;
        p.part_out = reinterpret_cast<float*>(ws + pl.many_out);
        p.part_ml = reinterpret_cast<float*>(ws + pl.many_ml);
        p.cuts = reinterpret_cast<AttnCut*>(ws + pl.many_cuts);
        e = launch_after_prepass(cache_attention_many_kernel<kDim, kBf16>, pl.many_grid, kManyThreads,
                                 (size_t)ManySmem<kDim>::bytes(p.requests), stream, mk, mv, p, cv);
        if (e == cudaSuccess && pl.many_grid > 1)
            e = launch_after_prepass(cache_attention_join_kernel<kManyRows, kDim, kBf16>,
                                     (pl.many_grid - 1) * (kManyRows / 16), 256, 0, stream, p);
    }
    return e;
}

}  // namespace blaze

using namespace blaze;

extern "C" int blazeCacheAttentionWorkspaceSize(const blazeKvCache* cache, const blazeCacheAttentionArgs* args, size_t* bytes) {
    if (!bytes) return ACLTENSOR_STATUS_INVALID_VALUE;
    DeviceContext* ctx = current_context();
    AttnPlan pl;
    const int st = plan_attention(cache, args, ctx ? ctx->sm_count : 148, &pl);
    if (st != ACLTENSOR_STATUS_SUCCESS) return st;
    *bytes = pl.total;
    return ACLTENSOR_STATUS_SUCCESS;
}

extern "C" int blazeCacheAttention(const blazeKvCache* cache, const blazeCacheAttentionArgs* a, void* stream_v) {
    DeviceContext* ctx = current_context();
    AttnPlan pl;
    const int st = plan_attention(cache, a, ctx ? ctx->sm_count : 148, &pl);
    if (st != ACLTENSOR_STATUS_SUCCESS) return st;
    if (a->requests == 0 || a->tokens == 0 || a->max_q == 0) return ACLTENSOR_STATUS_SUCCESS;
    auto aligned = [](const void* x, uintptr_t n) { return (reinterpret_cast<uintptr_t>(x) & (n - 1)) == 0; };
    if (!a->q || !a->out || !a->row_offsets || !a->kv_len || (a->max_blocks > 0 && !a->block_table))
        return ACLTENSOR_STATUS_INVALID_VALUE;
    if (!aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->lse, 4) || !aligned(a->row_offsets, 4) ||
        !aligned(a->kv_len, 4) || !aligned(a->block_table, 4) || (a->q_token_stride % 8) || (a->q_head_stride % 8) ||
        (a->out_token_stride % 8) || (a->out_head_stride % 8))
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    if (!a->workspace || a->workspace_bytes < pl.total) return ACLTENSOR_STATUS_INSUFFICIENT_WORKSPACE;
    if (!aligned(a->workspace, 256) || a->out == a->q) return ACLTENSOR_STATUS_INVALID_VALUE;
    if (!ctx) return ACLTENSOR_STATUS_NOT_INITIALIZED;
    if (ctx->cc_major != 10) return ACLTENSOR_STATUS_ARCH_MISMATCH;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);

    CUtensorMap mk, mv;
    const int box_rows = cache->block_size < kFewTokens ? cache->block_size : kFewTokens;
    if (!make_tmap_pages(&mk, cache->k, cache, box_rows) || !make_tmap_pages(&mv, cache->v, cache, box_rows))
        return ACLTENSOR_STATUS_INTERNAL_ERROR;

    const CacheView cv = cache_view(cache);
    CacheAttentionParams p;
    p.requests = a->requests;
    p.tokens = a->tokens;
    p.heads = a->heads;
    p.kv_heads = cache->kv_heads;
    p.group = a->heads / cache->kv_heads;
    p.block_shift = cv.block_shift;
    p.num_blocks = cache->num_blocks;
    p.max_blocks = a->max_blocks;
    p.max_q = a->max_q;
    p.max_kv = a->max_kv;
    p.causal = a->causal;
    p.window = a->window >= a->max_kv ? 0 : a->window;      // (wider than any request: none)
    p.scale_log2 = a->scale * kLog2E;
    p.q = a->q;
    p.q_token_stride = a->q_token_stride;
    p.q_head_stride = a->q_head_stride;
    p.out = a->out;
    p.out_token_stride = a->out_token_stride;
    p.out_head_stride = a->out_head_stride;
    p.lse = static_cast<float*>(a->lse);
    p.row_offsets = static_cast<const int*>(a->row_offsets);
    p.kv_len = static_cast<const int*>(a->kv_len);
    p.table = static_cast<const int*>(a->block_table);
    p.table_stride = a->table_stride;
    p.k_scale = cv.k_scale;
    p.v_scale = cv.v_scale;
    p.scale_stride = cv.scale_stride;
    p.status = ctx->status_word;
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    const bool bf16 = a->q_type == BLAZE_OUT_BF16;
    auto launch = cache->head_dim == 128 ? (bf16 ? launch_attention<128, true> : launch_attention<128, false>)
                                         : (bf16 ? launch_attention<64, true> : launch_attention<64, false>);
    return status_of(launch(mk, mv, p, cv, pl, ws, stream));
}
