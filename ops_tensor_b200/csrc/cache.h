// Internal declarations of the paged-cache kernels (cache.cu, cache_attention.cu).
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

#include "blaze_b200.h"

namespace blaze {

// The checks every entry point makes of the cache it is given; an acltensorStatus_t.
int check_kv_cache(const blazeKvCache* c);

struct CacheView {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    long long block_stride, head_stride, token_stride, scale_stride;
    int num_blocks, block_size, block_shift, kv_heads;
};
CacheView cache_view(const blazeKvCache* c);

}  // namespace blaze
