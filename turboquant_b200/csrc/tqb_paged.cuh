// What the files of the paged cache share.
#pragma once
#include <math.h>

#include <atomic>

#include "tqb_common.cuh"

namespace tqb {

// Status of a layer's description (tqb_paged_layer).
int check_paged_layer(const tqb_paged_layer* l);

// src/cache/wht_tensor.rs:29-35,43: rotation_fwd[0][j] * sqrt(32), all in f32
inline float block_sign_magnitude() {
    volatile float inv = 1.0f / sqrtf(32.0f);
    volatile float s = sqrtf(32.0f);
    return inv * s;
}

// More than 48 KB of shared memory, the static part included, is a property of the kernel on a device: set once for each, to
// `most` bytes (0: `bytes`, which is then the same in every call).
template <auto* KERNEL>
int allow_shared(int bytes, int most = 0) {
    static std::atomic<unsigned long long> configured{0};
    if (bytes <= 32 * 1024) return TQB_OK;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
    if (dev >= 0 && ((configured.load(std::memory_order_acquire) >> dev) & 1ull)) return TQB_OK;
    const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, most > bytes ? most : bytes);
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return TQB_ERR_CUDA;
    }
    if (dev >= 0) configured.fetch_or(1ull << dev, std::memory_order_release);
    return TQB_OK;
}

}  // namespace tqb
