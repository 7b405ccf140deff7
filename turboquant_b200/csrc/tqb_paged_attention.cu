// Attention of one new token of each request over the paged packed cache.
//
// A stored block decodes to k = |s| H (sigma .* c[code]) / sqrt(32) with the symmetric 32-point Hadamard matrix H, so
// <q, k> = |s| <sigma .* H q / sqrt(32), c[code]>: queries are rotated once, keys and values stay codes times scales, the
// sum over values is kept in the rotated domain and one inverse rotation is applied to the result.
#include "tqb_common.cuh"
#include "tqb_paged.cuh"
#include "tqb_paged_work.cuh"

namespace tqb {
namespace {

// One token a warp at a time, one lane a dim of every block, all in f32: f32 queries (whose precision the 16-bit weights of
// the tensor-core kernel would lose), and layers without pages.
template <int NB, int BITS>
__global__ void __launch_bounds__(kWorkThreads) paged_simple_kernel(const __grid_constant__ PagedArgs a) {
    constexpr int D = NB * 32;
    __shared__ float s_cent[16];
    __shared__ Fragments s_frag;
    extern __shared__ __align__(16) float s_o[];   // [2 kWorkWarps][kSegHeads][D]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < 16) s_cent[tid] = a.cent[tid];
    if (tid < 2 * kWorkWarps) s_frag.used[tid] = 0;
    WorkLine line(a);   // (its barriers stand before the first use of what is set above)
    const int page_mask = (1 << a.page_shift) - 1;
    Segment s;
    while (line.next(s)) {
        float q[kSegHeads][NB], o[kSegHeads][NB], m[kSegHeads], l[kSegHeads];
#pragma unroll
        for (int h = 0; h < kSegHeads; ++h) {
            m[h] = kNoScore;
            l[h] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                o[h][b] = 0.0f;
                q[h][b] = h < s.heads ? load_as_f32(a.q, a.q_dtype, (size_t)s.req * a.q_stride + (size_t)(s.head0 + h) * D + b * 32 + lane) : 0.0f;
                q[h][b] = wht32_across(q[h][b], lane) * (1.0f / sqrtf((float)kBlock)) * block_sign(lane, a.sign_mag) * a.qk_const;
            }
        }
        for (int t = s.t0; t < s.t1; ++t) {
            const int page = a.table[s.req * a.table_stride + (t >> a.page_shift)];
            if ((unsigned)page >= (unsigned)a.num_pages) continue;
            const size_t row = (((size_t)page * a.hkv + s.kvh) << a.page_shift) + (t & page_mask);
            float k[NB], v[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const size_t blk = row * NB + b;
                const int bit = BITS * lane;
                auto code = [&](const uint8_t* base) {
                    const uint8_t* p = base + blk * (4 * BITS) + (bit >> 3);
                    const unsigned w = p[0] | ((bit & 7) + BITS > 8 ? p[1] << 8 : 0);
                    return (w >> (bit & 7)) & ((1 << BITS) - 1);
                };
                k[b] = s_cent[code(a.kb)] * fabsf(f16_bits_to_f32(a.ks[blk]));
                v[b] = s_cent[code(a.vb)] * fabsf(f16_bits_to_f32(a.vs[blk]));
            }
#pragma unroll
            for (int h = 0; h < kSegHeads; ++h) {
                if (h >= s.heads) break;
                float x = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) x = fmaf(q[h][b], k[b], x);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
                const float mn = fmaxf(m[h], x), keep = exp2_fast(m[h] - mn), p = exp2_fast(x - mn);
                m[h] = mn;
                l[h] = fmaf(l[h], keep, p);
#pragma unroll
                for (int b = 0; b < NB; ++b) o[h][b] = fmaf(o[h][b], keep, p * v[b]);
            }
        }
        // (a whole segment's outputs pass through the slot of the warp's last one)
        const int slot = 2 * warp + (s.begins ? 1 : 0);
#pragma unroll
        for (int h = 0; h < kSegHeads; ++h) {
#pragma unroll
            for (int b = 0; b < NB; ++b) s_o[(slot * kSegHeads + h) * D + b * 32 + lane] = o[h][b];
            if (!s.whole() && lane == 0) {
                s_frag.m[slot][h] = m[h];
                s_frag.l[slot][h] = l[h];
            }
        }
        if (!s.whole() && lane == 0) {
            s_frag.seg[slot] = s;
            s_frag.used[slot] = 1;
        }
        __syncwarp();
        if (s.whole()) {
            const int quads = s.heads * (D / 4);
            for (int x0 = 0; x0 < quads; x0 += 32) {
                const int x = min(x0 + lane, quads - 1), hh = x / (D / 4);
                float L = l[0];
#pragma unroll
                for (int h = 1; h < kSegHeads; ++h) L = h == hh ? l[h] : L;
                write_quad(a.out, a.out_dtype, quad_at<NB>(a, s, x), x0 + lane < quads, reinterpret_cast<const float4*>(s_o + slot * kSegHeads * D)[x], L, a.sign_mag);
            }
            __syncwarp();
        }
    }
    finish<NB>(a, s_frag, [&](int c, int x) { return reinterpret_cast<const float4*>(s_o + c * kSegHeads * D)[x]; });
    write_empty<NB>(a);
}

template <int NB, int BITS>
int launch_simple(const PagedArgs& a, cudaStream_t s) {
    const int dyn = (int)sizeof(float) * 2 * kWorkWarps * kSegHeads * NB * 32;
    if (int st = allow_shared<paged_simple_kernel<NB, BITS>>(dyn)) return st;
    paged_simple_kernel<NB, BITS><<<148 * 4, kWorkThreads, dyn, s>>>(a);
    return check_launch(s);
}

size_t part_bytes(int head_dim) { return sizeof(float) * (size_t)kMaxCtas * 2 * kSegHeads * (2 + 2 + head_dim); }

}  // namespace
}  // namespace tqb

using namespace tqb;

extern "C" {

size_t tqb_paged_scratch_bytes(int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim) {
    if (num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    return TQB_PAGED_TICKET_BYTES + part_bytes(head_dim);
}

int tqb_paged_attention(const tqb_paged_layer* layer, const tqb_paged_attention_params* p, tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    int st = check_paged_layer(layer);
    if (st != TQB_OK) return st;
    if (!p) return TQB_ERR_NULL_POINTER;
    auto known = [](int t) { return t == TQB_F32 || t == TQB_F16 || t == TQB_BF16; };
    if (p->num_requests < 0 || p->num_q_heads <= 0 || p->max_blocks < 0 || p->table_stride < p->max_blocks || p->q_row_stride < 0 ||
        !known(p->q_dtype) || !known(p->out_dtype))
        return TQB_ERR_INVALID_ARGUMENT;
    if (p->num_q_heads % layer->num_kv_heads != 0) return TQB_ERR_DIMENSION_MISMATCH;
    if (p->q_row_stride != 0 && p->q_row_stride < (int64_t)p->num_q_heads * layer->head_dim) return TQB_ERR_INVALID_ARGUMENT;
    if (p->num_requests > TQB_PAGED_MAX_REQUESTS) return TQB_ERR_TOO_LARGE;
    if (p->num_requests == 0) return TQB_OK;
    if (!p->q || !p->out || !p->kv_lens || !p->scratch || (!p->block_table && p->max_blocks > 0)) return TQB_ERR_NULL_POINTER;
    const int64_t elem = p->q_dtype == TQB_F32 ? 4 : 2;
    if ((uintptr_t)p->q % 16 != 0 || (p->q_row_stride * elem) % 16 != 0 || (uintptr_t)p->out % 16 != 0 || (uintptr_t)p->scratch % 16 != 0 ||
        (uintptr_t)p->block_table % 4 != 0 || (uintptr_t)p->kv_lens % 4 != 0)
        return TQB_ERR_MISALIGNED;
    if (p->scratch_bytes < tqb_paged_scratch_bytes(p->num_q_heads, layer->num_kv_heads, layer->head_dim)) return TQB_ERR_INVALID_ARGUMENT;
    Codebook cb;
    if (!block_codebook(layer->bits, TQB_MAXNORM, cb)) return TQB_ERR_UNSUPPORTED_BITS;
    PagedArgs a{};
    a.q = p->q;
    a.out = p->out;
    a.kb = layer->k_indices;
    a.ks = layer->k_scales;
    a.vb = layer->v_indices;
    a.vs = layer->v_scales;
    a.table = p->block_table;
    a.lens = p->kv_lens;
    a.tickets = reinterpret_cast<unsigned*>(p->scratch);
    a.part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(p->scratch) + TQB_PAGED_TICKET_BYTES);
    a.round_ml = a.part_ml + (size_t)kMaxCtas * 2 * kSegHeads * 2;
    a.part_out = a.round_ml + (size_t)kMaxCtas * 2 * kSegHeads * 2;
    a.q_stride = p->q_row_stride != 0 ? p->q_row_stride : (long long)p->num_q_heads * layer->head_dim;
    a.table_stride = p->table_stride;
    a.requests = p->num_requests;
    a.max_blocks = p->max_blocks;
    const int64_t max_len = (int64_t)p->max_blocks * layer->page_size;
    a.max_len = (int)(max_len < 0x7fffff00 ? max_len : 0x7fffff00);   // (whole groups stay below 2^31)
    while ((1 << a.page_shift) < layer->page_size) ++a.page_shift;
    a.num_pages = layer->num_pages;
    a.hkv = layer->num_kv_heads;
    a.group = p->num_q_heads / layer->num_kv_heads;
    a.splits = (a.group + kSegHeads - 1) / kSegHeads;
    a.vheads = a.hkv * a.splits;
    // (below 2^30 units the quotients of divide() stay below 2^21)
    auto units = [&](int shift) { return (double)a.requests * (kOpenCost + 1 + (double)((a.max_len / kRunTokens) >> shift)) * a.vheads; };
    while (units(a.unit_shift) >= 1073741824.0 && a.unit_shift < 24) ++a.unit_shift;
    if (units(a.unit_shift) >= 1073741824.0) return TQB_ERR_TOO_LARGE;
    a.q_dtype = p->q_dtype;
    a.out_dtype = p->out_dtype;
    a.qk_const = p->softmax_scale * 1.4426950408889634f;
    a.sign_mag = block_sign_magnitude();
    for (int i = 0; i < 16; ++i) a.cent[i] = cb.c[i];
    cudaStream_t s = as_stream(stream);
    if (p->q_dtype != TQB_F32 && layer->num_pages > 0) return launch_paged_mma(a, layer->head_dim, layer->bits, s);
    switch (layer->head_dim * 10 + layer->bits) {
        case 643: return launch_simple<2, 3>(a, s);
        case 644: return launch_simple<2, 4>(a, s);
        case 1283: return launch_simple<4, 3>(a, s);
        case 1284: return launch_simple<4, 4>(a, s);
        case 2563: return launch_simple<8, 3>(a, s);
        default: return launch_simple<8, 4>(a, s);
    }
}

}  // extern "C"
