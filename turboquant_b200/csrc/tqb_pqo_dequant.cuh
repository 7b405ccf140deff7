// One 32-block of a one-codebook cache format dequantized by ONE thread: the body of block_dequantize_lane_kernel, shared with
// the paged cache.  Operations and order of polar_dequantize (src/cache/quantize_tensor.rs:179-220): centroid times signed
// magnitude, butterfly, 1 / sqrt(32), scale.
#pragma once
#include "tqb_f32x2.cuh"
#include "tqb_pqo_quant.cuh"

namespace tqb {

// [sign][code][lane] table of centroid times +-sign magnitude: 32 different banks a look-up, the sign of an element is an
// immediate offset.
template <int BITS>
struct DequantTable {
    static constexpr int kCodes = 1 << BITS, kBytes = kCodes * 128;   // bytes of one sign's table
};
template <int BITS>
__device__ __forceinline__ void build_dequant_table(const Codebook& cb, float sign_mag, unsigned char* tab, int tid, int nthreads) {
    using D = DequantTable<BITS>;
#pragma unroll 4
    for (int i = tid; i < D::kCodes * 32; i += nthreads) {
        const int code = i >> 5;
        const float v = cb.c[code < cb.n ? code : cb.n - 1] * sign_mag;
        reinterpret_cast<float*>(tab)[i] = v;
        reinterpret_cast<float*>(tab)[i + D::kCodes * 32] = -v;
    }
}

// w: the block's packed codes; as: (|scale|, |scale|); tab: the table, in shared memory; lane4: 4 * lane.  (The table's address is
// added to the row's, as a constant of the load: it need not be a multiple of the table's size.)
template <int BITS>
__device__ __forceinline__ void dequantize_values(const uint32_t (&w)[4], F2 as, const unsigned char* tab, uint32_t lane4, float (&v)[32]) {
    using D = DequantTable<BITS>;
    const F2 inv_sqrt = f2(1.0f / sqrtf((float)kBlock));
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        // the code moved to bits 7.. (its row of 128 bytes), the lane's bank below it
        const int k = (BITS * i) >> 5, sh = (BITS * i) & 31;
        const uint32_t m = sh < 7 ? w[k] << (7 - sh) : (sh + BITS <= 32 ? w[k] >> (sh - 7) : __funnelshift_r(w[k], w[k < 3 ? k + 1 : 3], sh - 7));
        const float* const row = reinterpret_cast<const float*>(tab + ((m & ((D::kCodes - 1) << 7)) | lane4));
        v[i] = row[((kSignMask >> i) & 1u) ? D::kBytes / 4 : 0];
    }
    F2 p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = f2(v[i], v[i + 16]);
    butterfly32_pairs(p);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 t = halves(mul2(mul2(p[i], inv_sqrt), as));
        v[i] = t.x;
        v[i + 16] = t.y;
    }
}

}  // namespace tqb
