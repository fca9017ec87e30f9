// Internal C++ declarations shared by the kernel translation units and the C-ABI layer.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

#include "cann_ops_tensor_types.h"

namespace blaze {

struct DeviceContext {
    int device = -1;
    int sm_count = 0;
    int cc_major = 0, cc_minor = 0;
    int* status_word = nullptr;     // device int, zero while no kernel wait has given up
};

// Per-device context of the current device (created on first use; thread-safe).  nullptr if no usable device.
DeviceContext* current_context();

// A launch's outcome as an acltensorStatus_t; clears the error.
inline int status_of(cudaError_t e) {
    if (e == cudaSuccess) return ACLTENSOR_STATUS_SUCCESS;
    cudaGetLastError();
    return ACLTENSOR_STATUS_EXECUTION_FAILED;
}

inline size_t round256(size_t x) { return (x + 255) & ~size_t(255); }

// cuTensorMapEncodeTiled, looked up through the runtime (the library does not link the driver); nullptr if missing.
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn();

// Launch of a kernel behind another one in its stream with programmatic stream serialisation: its blocks may set
// themselves up while the kernel before is still running, and wait for it (griddepcontrol.wait) before they touch
// memory.  Every block of such a kernel executes that wait before it ends, so that the kernel behind this one, which
// waits for this one alone, comes after the kernel before it as well.
template <class... KArgs, class... Args>
inline cudaError_t launch_after_prepass(void (*kernel)(KArgs...), int grid, int block, size_t smem, cudaStream_t stream,
                                        const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3((unsigned)block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Bytes of the re-tiled scale-factor array for `rows` x K with tiles of `tile_rows` rows, every 512-byte block
// stored `replicas` times in a row.
inline long long sf_tiled_bytes(int rows, int K, int tile_rows, int replicas = 1) {
    const long long tiles = (rows + tile_rows - 1) / tile_rows;
    const long long k_steps = (K + 127) / 128;
    const long long atoms = (tile_rows + 127) / 128;
    return tiles * k_steps * atoms * replicas * 512;
}

// `elem`: 0 = E4M3, 1 = packed E2M1, 2 = E5M2.
cudaError_t launch_quant_mx(const float* x, long long ldx, int rows, int K, int elem, uint8_t* codes,
                            long long ldc_bytes, uint8_t* scales, int sm_count, cudaStream_t stream);
cudaError_t launch_quant_fp8_1x128(const float* x, long long ldx, int rows, int K, uint8_t* codes, long long ldc,
                                   float* scales, int sm_count, cudaStream_t stream);
cudaError_t launch_quant_fp8_128x128(const float* w, long long ldw, int N, int K, uint8_t* codes, long long ldc,
                                     float* scales, int sm_count, cudaStream_t stream);
// `zero_ptr` / `zero_words`: 32-bit words the same kernel also clears (the stream-K flags of the GEMM that follows).
cudaError_t launch_sf_retile(const uint8_t* in, int rows, int K, int tile_rows, int replicas, uint8_t* out,
                             int sm_count, cudaStream_t stream, int* zero_ptr = nullptr, int zero_words = 0);
cudaError_t launch_e2m1_expand(const uint8_t* in, long long ld_in, int rows, int K, uint8_t* out, long long ld_out,
                               int sm_count, cudaStream_t stream);
// Pre-pass for a B stored [K][N] (N contiguous): its transpose [N][K] and its scales as rows [N][ceil(K/64)*2].
cudaError_t launch_transpose_bytes(const uint8_t* in, long long ld_in, int K, int N, uint8_t* out, long long ld_out,
                                   cudaStream_t stream);
cudaError_t launch_scale_pairs_to_rows(const uint8_t* in, int N, int K, uint8_t* out, int sm_count, cudaStream_t stream);
cudaError_t launch_add_f32(const float* a, const float* c, float* d, long long n, int sm_count, cudaStream_t stream);

}  // namespace blaze
