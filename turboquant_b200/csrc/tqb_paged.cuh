// What the files of the paged cache share.
#pragma once
#include <math.h>

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

}  // namespace tqb
