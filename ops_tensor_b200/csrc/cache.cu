// The paged 8-bit key / value cache: the step's block tables and slot maps, and the quantising store.
//
//   cache_assign   block tables, slots, positions, row offsets and lengths of a step from the requests' lengths
//   cache_store    bf16 / half keys and values -> E4M3 codes, one power-of-two scale per (block, head)
//
// The rules of both are spelled out at the entry points in include/blaze_b200.h.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <type_traits>

#include "cache.h"
#include "cann_ops_tensor_types.h"
#include "launch.h"
#include "ptx.cuh"

namespace blaze {

// ---------------------------------------------------------------------------------------------------- assign

constexpr int kAssignThreads = 1024;
constexpr int kAssignMaxRequests = 8192;
constexpr uint32_t kDeniedBit = 0x80000000u;

struct CacheAssignParams {
    int requests, block_size, block_shift, max_blocks, max_tokens, free_capacity;
    const int* cached_len;
    const int* new_len;
    int* table;
    long long table_stride;
    int* free_blocks;
    const int* free_count;
    int* free_count_out;
    int* row_offsets;
    int* kv_len;
    long long* slots;
    int* positions;
    int* denied;
    int write_lists;     // slots, positions, row offsets, table and stack
    int write_lengths;   // kv_len, free_count_out, denied
};

// Exclusive sum over the block's threads; `total` gets the sum of all.  Two barriers; safe to call again at once.
__device__ __forceinline__ long long block_exclusive_sum(long long x, long long* warp_sums, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    long long w = lane < (int)(blockDim.x >> 5) ? warp_sums[lane] : 0;
    long long winc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, winc, o);
        if (lane >= o) winc += y;
    }
    const long long before = __shfl_sync(0xffffffffu, winc - w, warp);
    total = __shfl_sync(0xffffffffu, winc, 31);
    __syncthreads();
    return before + inc - x;
}

// Last index i in [0, n) with start[i] <= x, for start not falling and start[0] <= x.
__device__ __forceinline__ int last_at_or_below(const int* start, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// Integer work, a few bytes per token: bound by latency (256 requests of one token, one block: 5.8 us) and, for
// prompts, by the binary search and the table load of each row (1000 requests, 640k rows, 148 blocks: 14.6 us, 0.6
// TB/s).  Every block makes the sums over all requests for itself in shared memory (8 bytes read per request, out of L2
// after the first), so blocks need nothing from one another: blocks popped from the stack are found by their number
// from the top, a popped block that an ended request gives back in the same call through the sum over the given-back
// blocks.  Reads and writes do not meet: the stack is read below free_count and written at or above it, table rows are
// read of one set of requests (old entries) and written for another (new entries).  The lengths, which may be updated
// in place, are written by a block that has read them all: the only one, or a second launch (`write_lists` = 0).
__global__ void __launch_bounds__(kAssignThreads) cache_assign_kernel(const CacheAssignParams p) {
    extern __shared__ int assign_smem[];
    __shared__ long long warp_sums[32];
    const int R = p.requests;
    int* row_start = assign_smem;                 // packed rows before request r
    int* need_start = row_start + R;              // blocks popped before request r
    int* back_start = need_start + R;             // blocks given back before request r
    uint32_t* old_len = reinterpret_cast<uint32_t*>(back_start + R);     // cached tokens | denied
    const int tid = threadIdx.x;

    grid_launch_dependents();
    grid_dependency_wait();
    const int capacity = p.max_blocks << p.block_shift;          // tokens that a row of the table can name
    const int per = (R + kAssignThreads - 1) / kAssignThreads;   // consecutive requests of this thread, at most 8
    const int r0 = min(R, tid * per), r1 = min(R, r0 + per);
    const int free_count = min(max(*p.free_count, 0), p.free_capacity);
    int news[8], olds[8];
    long long rows = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (r0 + j < r1) {
            news[j] = p.new_len[r0 + j];
            olds[j] = min(max(p.cached_len[r0 + j], 0), capacity);
            rows += max(news[j], 0);
        }
    }
    long long all_rows, all_need_back;
    long long row = block_exclusive_sum(rows, warp_sums, all_rows);
    // blocks needed in the high word, given back in the low one: both sums are below 2^31
    long long need_back = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (r0 + j < r1) {
            const int have = (olds[j] + p.block_size - 1) >> p.block_shift;
            row_start[r0 + j] = (int)min(row, (long long)p.max_tokens);
            bool fits = true;
            if (news[j] < 0) {
                need_back += have;
            } else {
                const long long end = (long long)olds[j] + news[j];
                row += news[j];
                fits = end <= capacity && (news[j] == 0 || row <= p.max_tokens);
                const int need = fits ? (int)((end + p.block_size - 1) >> p.block_shift) - have : 0;
                need_back += (long long)need << 32;
            }
            old_len[r0 + j] = (uint32_t)olds[j] | (fits ? 0u : kDeniedBit);
        }
    }
    long long nb = block_exclusive_sum(need_back, warp_sums, all_need_back);
    const int returned = (int)(all_need_back & 0xFFFFFFFFll);
    const long long top = (long long)free_count + returned;      // height of the stack with the returned blocks on it
    long long popped_denied = 0;                                 // largest served sum of needs; denied requests above it
    int my_popped = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (r0 + j < r1) {
            const int r = r0 + j;
            const int have = (olds[j] + p.block_size - 1) >> p.block_shift;
            need_start[r] = (int)(nb >> 32);
            back_start[r] = (int)(nb & 0xFFFFFFFFll);
            bool denied = (old_len[r] & kDeniedBit) != 0;
            if (news[j] < 0) {
                nb += have;
            } else if (!denied) {
                const int need = (int)(((long long)olds[j] + news[j] + p.block_size - 1) >> p.block_shift) - have;
                nb += (long long)need << 32;
                if (need > 0) {
                    if ((nb >> 32) > top) { denied = true; old_len[r] |= kDeniedBit; } else my_popped = (int)(nb >> 32);
                }
            }
            popped_denied += denied ? 1 : 0;
            if (p.write_lengths && blockIdx.x == 0) {
                // (every length has been read into registers before the barriers above)
                p.kv_len[r] = news[j] < 0 ? 0 : (denied ? olds[j] : olds[j] + news[j]);
            }
        }
    }
    // the needs of served requests are a prefix of all needs, so the largest served sum is what the stack gives away
    __shared__ int s_popped, s_denied;
    if (tid == 0) { s_popped = 0; s_denied = 0; }
    __syncthreads();
    if (my_popped > 0) atomicMax(&s_popped, my_popped);
    if (popped_denied > 0) atomicAdd(&s_denied, (int)popped_denied);
    __syncthreads();
    const int popped = s_popped;
    const int stack_left = (int)(top - popped);
    if (p.write_lengths && blockIdx.x == 0 && tid == 0) {
        *p.free_count_out = min(stack_left, p.free_capacity);
        if (p.denied) *p.denied = s_denied;
    }
    if (!p.write_lists) return;

    auto given_back = [&](int j) -> int {                         // j-th block that comes back in this call
        const int r = last_at_or_below(back_start, R, j);
        return p.table[(long long)r * p.table_stride + (j - back_start[r])];
    };
    auto from_top = [&](int n) -> int {                           // n-th block popped
        const int at = (int)(top - 1 - n);
        return at < free_count ? p.free_blocks[at] : given_back(at - free_count);
    };
    const int threads = gridDim.x * kAssignThreads;
    const int t0 = blockIdx.x * kAssignThreads + tid;
    const int total_rows = (int)min(all_rows, (long long)p.max_tokens);
    for (int r = t0; r <= R; r += threads) p.row_offsets[r] = r < R ? row_start[r] : total_rows;
    // new table entries: the n-th popped block
    for (int n = t0; n < popped; n += threads) {
        const int r = last_at_or_below(need_start, R, n);
        const int have = (int)((old_len[r] & ~kDeniedBit) + p.block_size - 1) >> p.block_shift;
        p.table[(long long)r * p.table_stride + have + (n - need_start[r])] = from_top(n);
    }
    // returned blocks that stay on the stack
    for (int at = free_count + t0; at < min(stack_left, p.free_capacity); at += threads)
        p.free_blocks[at] = given_back(at - free_count);
    // slots and positions of the packed rows
    for (int t = t0; t < p.max_tokens; t += threads) {
        long long slot = -1;
        int pos = -1;
        if (t < total_rows) {
            const int r = last_at_or_below(row_start, R, t);
            const uint32_t ol = old_len[r];
            const int old = (int)(ol & ~kDeniedBit);
            const int at = t - row_start[r];
            pos = old + at;
            if (!(ol & kDeniedBit)) {
                const int col = pos >> p.block_shift;
                const int have = (old + p.block_size - 1) >> p.block_shift;
                const int block = col < have ? p.table[(long long)r * p.table_stride + col]
                                             : from_top(need_start[r] + col - have);
                slot = (long long)block * p.block_size + (pos & (p.block_size - 1));
            }
        }
        p.slots[t] = slot;
        if (p.positions) p.positions[t] = pos;
    }
}

// ---------------------------------------------------------------------------------------------------- store

constexpr int kScaleMinExp = -64, kScaleMaxExp = 120;
constexpr int kStoreWarps = 4;

struct CacheStoreParams {
    CacheView cache;
    const void* x[2];                        // rows of K and of V
    long long token_stride[2], head_stride[2];
    const long long* slots;
    int tokens;
    long long slot_count;
    int window;                              // rows of the call whose runs one block takes
};

template <bool kBf16>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
    if constexpr (kBf16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        a = f.x;
        b = f.y;
    }
}

// Largest finite magnitude of the two 16-bit values of each word, as their bit pattern (bit patterns of non-negative
// floats order like the floats; infinities and NaNs count as zero).
template <bool kBf16>
__device__ __forceinline__ uint32_t max_finite(uint32_t m, uint32_t w) {
    constexpr uint32_t kInf = kBf16 ? 0x7F80u : 0x7C00u;
    const uint32_t lo = w & 0x7FFFu, hi = (w >> 16) & 0x7FFFu;
    m = max(m, lo < kInf ? lo : 0u);
    return max(m, hi < kInf ? hi : 0u);
}

// The smallest power of two with amax <= 448 * 2^e: 448 = 1.75 * 2^8, so e is amax's exponent less 8, one more when
// its mantissa is above 1.75.
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t b = __float_as_uint(amax);
    int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    if (amax == 0.0f) e = kScaleMinExp;
    e = min(max(e, kScaleMinExp), kScaleMaxExp);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// codes -> codes of the same values under a scale `ratio` times the old one's inverse
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
    float f[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&r));
        f[2 * h] = v.x * ratio;
        f[2 * h + 1] = v.y * ratio;
    }
    return cvt_e4m3x4_sat(f[0], f[1], f[2], f[3]);
}

// The magnitudes' maxima of the words' low and high halves, infinities and NaNs among them (they come out on top).
__device__ __forceinline__ uint32_t max_any(uint32_t m, const uint4& v) {
    m = __vmaxu2(m, v.x & 0x7FFF7FFFu);
    m = __vmaxu2(m, v.y & 0x7FFF7FFFu);
    m = __vmaxu2(m, v.z & 0x7FFF7FFFu);
    return __vmaxu2(m, v.w & 0x7FFF7FFFu);
}
template <bool kBf16>
__device__ __forceinline__ bool any_not_finite(uint32_t m) {
    constexpr uint32_t kInf = kBf16 ? 0x7F80u : 0x7C00u;
    return (m & 0xFFFFu) >= kInf || (m >> 16) >= kInf;
}

// Eight 16-bit inputs -> eight codes under a scale: x * inv where 1 / scale is exact, else a division.
template <bool kBf16, bool kExact>
__device__ __forceinline__ uint2 encode8(const uint4& v, float inv, float scale) {
    float f[8];
    unpack2<kBf16>(v.x, f[0], f[1]);
    unpack2<kBf16>(v.y, f[2], f[3]);
    unpack2<kBf16>(v.z, f[4], f[5]);
    unpack2<kBf16>(v.w, f[6], f[7]);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = kExact ? f[i] * inv : __fdiv_rn(f[i], scale);
    return make_uint2(cvt_e4m3x4_sat(f[0], f[1], f[2], f[3]), cvt_e4m3x4_sat(f[4], f[5], f[6], f[7]));
}

// A run is what neighbouring rows of the call put into one block; it is taken up for one head of K or of V at a time.
// Runs of more than kStoreShort rows are shared by the block's four warps: every lane holds its 16-byte pieces of up to
// eight rows from the one read (a block of 64 tokens then needs no second), the largest magnitude goes through shared
// memory.  Shorter runs (a decode step's single rows) go to one warp each.
// Bytes: 4 read and 2 written per (token, head, dim) of K and V together.  26k rows of 8 heads of 128: 46 us, 3.4 TB/s, bound
// by the dependent loads of a run (slots, rows, old scale) at the 32 warps of an SM that 64 registers allow (64 bytes spilled).
// 128 single rows: 6.1 us, latency.  Runs by one warp each / shared: of 2 rows (200 in all) 4.8 / 5.7 us, of 4 (400) 6.3 / 7.1,
// of 8 (800) 6.7 / 8.2, of 12 (480) the same; but with a limit of 16 the short runs at the ends of prompts hold the others
// up (4800 rows of four 11.9 us against 9.7).
constexpr int kStoreShort = 4;

template <int kDim, bool kBf16>
__global__ void __launch_bounds__(kStoreWarps * 32, 8) cache_store_kernel(const CacheStoreParams p) {
    constexpr int kLanesPerRow = kDim / 8;               // 16 bytes of input, 8 of codes per lane
    constexpr int kRowsPerLoad = 32 / kLanesPerRow;
    constexpr int kBatch = 8;
    __shared__ uint32_t warp_max[2][kStoreWarps];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / kLanesPerRow;                 // row of a load that this lane has a part of
    const int col = (lane % kLanesPerRow) * 8;
    // heads of K and V beside one another, so that what runs together reads whole rows of the input
    const int units = 2 * p.cache.kv_heads;
    const int win = blockIdx.x / units;
    const int unit = blockIdx.x - win * units;
    const int which = unit >= p.cache.kv_heads ? 1 : 0, head = unit - which * p.cache.kv_heads;
    const int w0 = win * p.window;
    const int w1 = min(p.tokens, w0 + p.window);
    const uint16_t* x = static_cast<const uint16_t*>(p.x[which]) + head * p.head_stride[which] + col;
    const long long row_stride = p.token_stride[which];
    uint8_t* codes = (which ? p.cache.v : p.cache.k) + head * p.cache.head_stride + col;
    float* scales = (which ? p.cache.v_scale : p.cache.k_scale) + head;
    const int shift = p.cache.block_shift;

    auto block_of = [&](int t) -> long long {            // block that row t goes to, or -1
        const long long s = p.slots[t];
        return (s < 0 || s >= p.slot_count) ? -1 : (s >> shift);
    };
    auto load = [&](int row, int end) -> uint4 {
        return row < end ? *reinterpret_cast<const uint4*>(x + (long long)row * row_stride) : make_uint4(0, 0, 0, 0);
    };
    int turn = 0;                                        // short runs of the window, dealt to the warps in turn
    int shared_runs = 0;
    for (int base = w0; base < w1; base += 32) {
        const int t = base + lane;
        const long long mine = t < w1 ? block_of(t) : -1;
        long long before = __shfl_up_sync(0xffffffffu, mine, 1);
        if (lane == 0) before = base > 0 ? block_of(base - 1) : -1;
        uint32_t starts = __ballot_sync(0xffffffffu, t < w1 && mine >= 0 && mine != before);
        while (starts) {
            const int first = __ffs(starts) - 1;
            starts &= starts - 1;
            const int a = base + first;
            const long long block = __shfl_sync(0xffffffffu, mine, first);
            // the run's end, and its lowest row within the block
            int b = a, low = p.cache.block_size;
            bool twice = false;                          // rows out of order: a slot may be named twice
            for (;;) {
                const int u = b + lane;
                const long long s = u < p.tokens ? p.slots[u] : -1;
                const bool in = s >= 0 && s < p.slot_count && (s >> shift) == block;
                const uint32_t out = ~__ballot_sync(0xffffffffu, in);
                const int n = out ? __ffs(out) - 1 : 32;
                const int at = (int)(s & (p.cache.block_size - 1));
                low = min(low, (int)__reduce_min_sync(0xffffffffu, lane < n ? (unsigned)at : 0x7FFFFFFFu));
                const long long s_before = (lane < n && u > a) ? p.slots[u - 1] : s - 1;
                twice |= __any_sync(0xffffffffu, lane < n && s != s_before + 1);
                b += n;
                if (n < 32) break;
            }
            const bool shared = b - a > kStoreShort && !twice;
            if (!shared && (turn++ % kStoreWarps) != warp) continue;
            // this warp's rows: r0, r0 + step, ...; all that a lane loads at once is kept when it is all there is
            const int span = kRowsPerLoad * kBatch;
            const int step = shared ? span * kStoreWarps : span;
            const int r0 = shared ? a + warp * span : a;
            const bool kept = b - a <= step;
            uint4 v[kBatch];
            uint32_t m = 0;
            for (int r = r0; r < b; r += step) {
#pragma unroll
                for (int j = 0; j < kBatch; ++j) v[j] = load(r + j * kRowsPerLoad + sub, b);
#pragma unroll
                for (int j = 0; j < kBatch; ++j) m = max_any(m, v[j]);
            }
            if (__any_sync(0xffffffffu, any_not_finite<kBf16>(m))) {
                // rare: infinities and NaNs do not count
                m = 0;
                for (int r = r0 + sub; r < b; r += step) {
#pragma unroll 1
                    for (int j = 0; j < kBatch; ++j) {
                        const uint4 w = load(r + j * kRowsPerLoad, b);
                        m = max_finite<kBf16>(max_finite<kBf16>(max_finite<kBf16>(max_finite<kBf16>(m, w.x), w.y), w.z), w.w);
                    }
                }
            } else {
                m = max(m & 0xFFFFu, m >> 16);
            }
            m = __reduce_max_sync(0xffffffffu, m);
            float* scale_at = scales + block * p.cache.scale_stride;
            const float old = low > 0 ? *scale_at : 0.0f;
            if (shared) {
                uint32_t* wm = warp_max[shared_runs++ & 1];
                if (lane == 0) wm[warp] = m;
                __syncthreads();                         // (and every warp has read the old scale)
#pragma unroll
                for (int w = 0; w < kStoreWarps; ++w) m = max(m, wm[w]);
            }
            float amax, unused;
            unpack2<kBf16>(m, amax, unused);
            const float need = scale_for(amax);
            const float scale = old >= need ? old : need;
            // 1 / scale is exact for the powers of two that this store writes; another scale is divided by
            const bool pow2 = (__float_as_uint(scale) & 0x7FFFFFu) == 0 && scale >= 0x1p-64f && scale <= 0x1p120f;
            const float inv = pow2 ? __uint_as_float((254u << 23) - __float_as_uint(scale)) : 0.0f;
            uint8_t* page = codes + block * p.cache.block_stride;
            if (scale != old && old > 0.0f) {
                const float ratio = old / scale;
                for (int r = sub + (shared ? warp * kRowsPerLoad : 0); r < low; r += kRowsPerLoad * (shared ? kStoreWarps : 1)) {
                    uint2* at = reinterpret_cast<uint2*>(page + (long long)r * p.cache.token_stride);
                    const uint2 w = *at;
                    *at = make_uint2(rescale4(w.x, ratio), rescale4(w.y, ratio));
                }
            }
            if (shared) {
                // slots rise one by one: row r goes to slot low + r - a
                auto put = [&](auto exact) {
                    for (int r = r0; r < b; r += step) {
                        if (!kept) {
#pragma unroll
                            for (int j = 0; j < kBatch; ++j) v[j] = load(r + j * kRowsPerLoad + sub, b);
                        }
                        uint8_t* at = page + (long long)(low + r + sub - a) * p.cache.token_stride;
#pragma unroll
                        for (int j = 0; j < kBatch; ++j) {
                            if (r + j * kRowsPerLoad + sub < b)
                                *reinterpret_cast<uint2*>(at + (long long)(j * kRowsPerLoad) * p.cache.token_stride) =
                                    encode8<kBf16, decltype(exact)::value>(v[j], inv, scale);
                        }
                    }
                };
                if (pow2) put(std::true_type{}); else put(std::false_type{});
                if (threadIdx.x == 0 && scale != old) *scale_at = scale;
            } else {
                for (int r = r0; r < b; r += kRowsPerLoad) {
                    const int row = r + sub;
                    const uint4 w = load(row, b);
                    const long long slot = row < b ? p.slots[row] : 0;
                    // rows that name a slot twice: the rows of one step are the only ones that could meet, and the last
                    // of them has to win
                    bool last = row < b;
#pragma unroll
                    for (int o = 1; o < kRowsPerLoad; ++o) {
                        const long long s = __shfl_down_sync(0xffffffffu, slot, o * kLanesPerRow);
                        if (sub + o < kRowsPerLoad && row + o < b && s == slot) last = false;
                    }
                    if (last)
                        *reinterpret_cast<uint2*>(page + (long long)(slot & (p.cache.block_size - 1)) * p.cache.token_stride) =
                            pow2 ? encode8<kBf16, true>(w, inv, scale) : encode8<kBf16, false>(w, inv, scale);
                    __syncwarp();                        // the next rows' stores come behind these
                }
                if (lane == 0 && scale != old) *scale_at = scale;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------- checks

static bool pointer_ok(const void* p, uintptr_t align) { return p && (reinterpret_cast<uintptr_t>(p) & (align - 1)) == 0; }

static int shift_of(int block_size) {
    switch (block_size) {
        case 16: return 4;
        case 32: return 5;
        case 64: return 6;
        case 128: return 7;
        default: return -1;
    }
}

int check_kv_cache(const blazeKvCache* c) {
    if (!c || c->struct_size < sizeof(blazeKvCache)) return ACLTENSOR_STATUS_INVALID_VALUE;
    if (c->num_blocks < 1 || c->kv_heads < 1) return ACLTENSOR_STATUS_INVALID_VALUE;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return ACLTENSOR_STATUS_INVALID_VALUE;
    if (c->elem != BLAZE_ELEM_E4M3 || shift_of(c->block_size) < 0 || (c->head_dim != 64 && c->head_dim != 128))
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    if (!pointer_ok(c->k, 16) || !pointer_ok(c->v, 16) || !pointer_ok(c->k_scale, 4) || !pointer_ok(c->v_scale, 4))
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    if (c->token_stride < c->head_dim || (c->kv_heads > 1 && c->head_stride < c->head_dim) ||
        (c->num_blocks > 1 && c->block_stride < c->head_dim) || c->scale_stride < c->kv_heads)
        return ACLTENSOR_STATUS_INVALID_VALUE;
    if ((c->token_stride % 16) || (c->kv_heads > 1 && c->head_stride % 16) || (c->num_blocks > 1 && c->block_stride % 16))
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    const int64_t limit = int64_t(1) << 40;              // strides that a tensor map can hold
    if (c->token_stride >= limit || c->head_stride >= limit || c->block_stride >= limit)
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    return ACLTENSOR_STATUS_SUCCESS;
}

CacheView cache_view(const blazeKvCache* c) {
    CacheView v;
    v.k = static_cast<uint8_t*>(c->k);
    v.v = static_cast<uint8_t*>(c->v);
    v.k_scale = static_cast<float*>(c->k_scale);
    v.v_scale = static_cast<float*>(c->v_scale);
    v.block_stride = c->num_blocks > 1 ? c->block_stride : 0;
    v.head_stride = c->kv_heads > 1 ? c->head_stride : 0;
    v.token_stride = c->token_stride;
    v.scale_stride = c->scale_stride;
    v.num_blocks = c->num_blocks;
    v.block_size = c->block_size;
    v.block_shift = shift_of(c->block_size);
    v.kv_heads = c->kv_heads;
    return v;
}

template <class K>
static cudaError_t allow_smem(K kernel, int bytes, bool (&done)[64]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (done[dev & 63]) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done[dev & 63] = true;
    return e;
}

}  // namespace blaze

using namespace blaze;

extern "C" int blazeCacheAssign(const blazeCacheAssignArgs* a, void* stream_v) {
    if (!a || a->struct_size < sizeof(blazeCacheAssignArgs)) return ACLTENSOR_STATUS_INVALID_VALUE;
    if (a->requests < 0 || a->max_blocks < 0 || a->max_tokens < 0 || a->free_capacity < 0 ||
        a->table_stride < a->max_blocks)
        return ACLTENSOR_STATUS_INVALID_VALUE;
    const int shift = shift_of(a->block_size);
    if (shift < 0 || a->requests > kAssignMaxRequests || ((int64_t)a->max_blocks << shift) > 0x7FFFFFFFll ||
        (int64_t)a->max_blocks * a->requests > 0x7FFFFFFFll)
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    if (!pointer_ok(a->free_count, 4) || !pointer_ok(a->free_count_out, 4) || !pointer_ok(a->row_offsets, 4))
        return ACLTENSOR_STATUS_INVALID_VALUE;
    if (a->requests > 0 && (!pointer_ok(a->cached_len, 4) || !pointer_ok(a->new_len, 4) || !pointer_ok(a->kv_len, 4)))
        return ACLTENSOR_STATUS_INVALID_VALUE;
    if ((a->requests > 0 && a->max_blocks > 0 && !pointer_ok(a->block_table, 4)) ||
        (a->free_capacity > 0 && !pointer_ok(a->free_blocks, 4)) || (a->max_tokens > 0 && !pointer_ok(a->slots, 8)) ||
        (reinterpret_cast<uintptr_t>(a->positions) & 3) || (reinterpret_cast<uintptr_t>(a->denied) & 3))
        return ACLTENSOR_STATUS_INVALID_VALUE;
    DeviceContext* ctx = current_context();
    if (!ctx) return ACLTENSOR_STATUS_NOT_INITIALIZED;
    if (ctx->cc_major != 10) return ACLTENSOR_STATUS_ARCH_MISMATCH;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);

    CacheAssignParams p;
    p.requests = a->requests;
    p.block_size = a->block_size;
    p.block_shift = shift;
    p.max_blocks = a->max_blocks;
    p.max_tokens = a->max_tokens;
    p.free_capacity = a->free_capacity;
    p.cached_len = static_cast<const int*>(a->cached_len);
    p.new_len = static_cast<const int*>(a->new_len);
    p.table = static_cast<int*>(a->block_table);
    p.table_stride = a->table_stride;
    p.free_blocks = static_cast<int*>(a->free_blocks);
    p.free_count = static_cast<const int*>(a->free_count);
    p.free_count_out = static_cast<int*>(a->free_count_out);
    p.row_offsets = static_cast<int*>(a->row_offsets);
    p.kv_len = static_cast<int*>(a->kv_len);
    p.slots = static_cast<long long*>(a->slots);
    p.positions = static_cast<int*>(a->positions);
    p.denied = static_cast<int*>(a->denied);

    static bool smem_done[64] = {};
    cudaError_t e = allow_smem(cache_assign_kernel, kAssignMaxRequests * 16, smem_done);
    if (e != cudaSuccess) return status_of(e);
    const size_t smem = (size_t)(a->requests > 0 ? a->requests : 1) * 16;
    const long long wanted = ((long long)a->max_tokens + kAssignThreads - 1) / kAssignThreads;
    const int grid = (int)(wanted < 1 ? 1 : (wanted > ctx->sm_count ? ctx->sm_count : wanted));
    const bool in_place = a->kv_len == a->cached_len || a->free_count_out == a->free_count;
    p.write_lists = 1;
    p.write_lengths = (grid == 1 || !in_place) ? 1 : 0;
    e = launch_after_prepass(cache_assign_kernel, grid, kAssignThreads, smem, stream, p);
    if (e == cudaSuccess && !p.write_lengths) {
        p.write_lists = 0;
        p.write_lengths = 1;
        e = launch_after_prepass(cache_assign_kernel, 1, kAssignThreads, smem, stream, p);
    }
    return status_of(e);
}

extern "C" int blazeCacheStore(const blazeKvCache* cache, const blazeCacheStoreArgs* a, void* stream_v) {
    const int st = check_kv_cache(cache);
    if (st != ACLTENSOR_STATUS_SUCCESS) return st;
    if (!a || a->struct_size < sizeof(blazeCacheStoreArgs) || a->tokens < 0) return ACLTENSOR_STATUS_INVALID_VALUE;
    if (a->in_type != BLAZE_OUT_BF16 && a->in_type != BLAZE_OUT_F16) return ACLTENSOR_STATUS_NOT_SUPPORTED;
    if (a->tokens == 0) return ACLTENSOR_STATUS_SUCCESS;
    if (!a->k || !a->v || !pointer_ok(a->slots, 8)) return ACLTENSOR_STATUS_INVALID_VALUE;
    if (!pointer_ok(a->k, 16) || !pointer_ok(a->v, 16) || (a->k_token_stride % 8) || (a->v_token_stride % 8) ||
        (a->k_head_stride % 8) || (a->v_head_stride % 8))
        return ACLTENSOR_STATUS_NOT_SUPPORTED;
    DeviceContext* ctx = current_context();
    if (!ctx) return ACLTENSOR_STATUS_NOT_INITIALIZED;
    if (ctx->cc_major != 10) return ACLTENSOR_STATUS_ARCH_MISMATCH;

    CacheStoreParams p;
    p.cache = cache_view(cache);
    p.x[0] = a->k;
    p.x[1] = a->v;
    p.token_stride[0] = a->k_token_stride;
    p.token_stride[1] = a->v_token_stride;
    p.head_stride[0] = a->k_head_stride;
    p.head_stride[1] = a->v_head_stride;
    p.slots = static_cast<const long long*>(a->slots);
    p.tokens = a->tokens;
    p.slot_count = (long long)cache->num_blocks * cache->block_size;
    // Rows per block: few where the call has too few for all SMs, many where each block would repeat the search for its runs.
    // 4 / 16 / 64 rows: 400 single rows 9.1 / 14.8 / 41 us; 1500 rows of a prompt 10.0 / 6.4 / 6.7; 4800 of four 23.7 / 12.0 / 9.7;
    // 26k of sixteen 128 / 58 / 47; but 4500 single rows 73 / 68 / 79.
    p.window = a->tokens >= 4096 ? 64 : (a->tokens >= 512 ? 16 : 4);
    const long long blocks = (long long)((a->tokens + p.window - 1) / p.window) * 2 * cache->kv_heads;
    if (blocks > 0x7FFFFFFFll) return ACLTENSOR_STATUS_NOT_SUPPORTED;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool bf16 = a->in_type == BLAZE_OUT_BF16;
    auto kernel = cache->head_dim == 128 ? (bf16 ? cache_store_kernel<128, true> : cache_store_kernel<128, false>)
                                         : (bf16 ? cache_store_kernel<64, true> : cache_store_kernel<64, false>);
    return status_of(launch_after_prepass(kernel, (int)blocks, kStoreWarps * 32, 0, stream, p));
}
