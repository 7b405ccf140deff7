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

// Queries in f32 (whose precision the 16-bit weights of the tensor-core kernel would lose), and layers without pages: everything
// in f32, on the FMA pipes.  A warp takes 32 tokens of its segment at a time:
//   scores   a lane a token: its codes' centroids from a table in shared memory (a copy for each bank) times the rotated queries,
//            [dim][head] in shared memory, four heads a read that all lanes share;
//   softmax  running maximum and sum, the maximum over the 32 lanes, weights to shared memory as [token][head];
//   values   a lane a dim of every block, token after token: centroid times |scale|, times the weight of each head.
// Bound: instructions, about 75 a token of a KV head for up to four query heads, 100 for eight (the copies are a tenth of the
// time).  A token at a time with its score summed over the lanes took 1,220 us instead of 178 for 64 requests of up to 8,192
// tokens, 8 KV heads of four query heads, head_dim 128.
constexpr int kStepTokens = 32;

template <int NB, int H, int BITS>
struct F32Plan {
    static constexpr int kD = NB * 32, kRow = 4 * BITS * NB;
    static constexpr int kQueries = kD * H * 4;                       // of a warp: [dim][head]; its last segment's outputs, later
    static constexpr int kCodes = kStepTokens * kRow;                 // of K, of V
    static constexpr int kWeights = kStepTokens * H * 4;
    static constexpr int kScales = kStepTokens * NB * 4;              // of K, of V
    static constexpr int kArea = kQueries + 2 * kCodes + kWeights + 2 * kScales;
    static constexpr int kWarpBytes = kArea + kQueries;               // and the outputs of its first segment, if others share it
    static constexpr int kBytes = kWorkWarps * kWarpBytes;
    static constexpr int kByShared = 228 * 1024 / (kBytes + 1024 + 4096), kByRegs = NB == 8 ? (H == 8 ? 2 : 3) : H == 8 ? 3 : 4;
    static constexpr int kCtas = kByShared < kByRegs ? kByShared : kByRegs;
    static_assert(kCtas >= 1 && kRow % 8 == 0, "an SM has no room for a CTA");
};

template <int BYTES>
__device__ __forceinline__ void copy_piece(void* dst, const void* src) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) cp_async16(to, src);
    else cp_async_ca<BYTES>(to, src);
}

// A token's NB scales as f32 magnitudes.
template <int NB>
__device__ __forceinline__ void scales_of(const uint16_t* from, bool live, float* to) {
    uint32_t w[NB / 2];
#pragma unroll
    for (int i = 0; i < NB / 2; ++i) w[i] = live ? __ldg(reinterpret_cast<const uint32_t*>(from) + i) : 0u;
#pragma unroll
    for (int i = 0; i < NB / 2; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        *reinterpret_cast<float2*>(to + 2 * i) = make_float2(fabsf(f.x), fabsf(f.y));
    }
}

template <int NB, int H, int BITS>
__global__ void __launch_bounds__(kWorkThreads, F32Plan<NB, H, BITS>::kCtas) paged_f32_kernel(const __grid_constant__ PagedArgs a) {
    using L = F32Plan<NB, H, BITS>;
    constexpr int D = L::kD, kPiece = L::kRow % 16 == 0 ? 16 : 8;
    __shared__ float s_cent[1 << BITS][32];
    __shared__ Fragments s_frag;
    extern __shared__ __align__(16) unsigned char s_dyn[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned char* const area = s_dyn + warp * L::kWarpBytes;
    float* const s_q = reinterpret_cast<float*>(area);                                          // [dim][head]
    unsigned char* const s_k = area + L::kQueries;                                              // [token] rows of codes
    unsigned char* const s_v = s_k + L::kCodes;
    float* const s_p = reinterpret_cast<float*>(s_v + L::kCodes);                               // [token][head]
    float* const s_ks = s_p + kStepTokens * H;                                                  // [token][block]
    float* const s_vs = s_ks + kStepTokens * NB;
    // outputs [H][D] of a fragment: that of the warp's last segment lies over its queries
    auto fragment = [&](int slot) { return reinterpret_cast<float*>(s_dyn + (slot >> 1) * L::kWarpBytes + ((slot & 1) ? 0 : L::kArea)); };
    for (int i = tid; i < (1 << BITS) * 32; i += kWorkThreads) s_cent[i >> 5][i & 31] = a.cent[i >> 5];
    if (tid < 2 * kWorkWarps) s_frag.used[tid] = 0;
    WorkLine line(a);   // (its barriers stand before the first use of what is set above)
    const int page_mask = (1 << a.page_shift) - 1;
    const unsigned char* const cent = reinterpret_cast<const unsigned char*>(&s_cent[0][lane]);
    auto centroid = [&](uint32_t at) { return *reinterpret_cast<const float*>(cent + (at & (((1u << BITS) - 1) << 7))); };   // code at bit 7
    Segment s;
    while (line.next(s)) {
        // ---- queries ----
#pragma unroll 1
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float q = h < s.heads ? load_as_f32(a.q, a.q_dtype, (size_t)known_row(a, s.req) * a.q_stride + (size_t)(s.head0 + h) * D + b * 32 + lane) : 0.0f;
                s_q[(b * 32 + lane) * H + h] = wht32_across(q, lane) * (1.0f / sqrtf((float)kBlock)) * block_sign(lane, a.sign_mag) * a.qk_const;
            }
        float o[H][NB], m[H], l[H];   // l: of the lane's tokens
#pragma unroll
        for (int h = 0; h < H; ++h) {
            m[h] = kNoScore;
            l[h] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) o[h][b] = 0.0f;
        }
#pragma unroll 1
        for (int t0 = s.t0; t0 < s.t1; t0 += kStepTokens) {
            // ---- a lane a token: codes and scales ----
            const int t = t0 + lane, last = s.t1 - t0 < kStepTokens ? s.t1 - t0 : kStepTokens;
            const int page = t < s.t1 ? a.table[s.req * a.table_stride + (t >> a.page_shift)] : -1;
            const bool live = (unsigned)page < (unsigned)a.num_pages;
            const size_t row = ((((size_t)(live ? page : 0) * a.hkv + s.kvh) << a.page_shift) + (t & page_mask));
            if (live) {
#pragma unroll
                for (int i = 0; i < L::kRow; i += kPiece) {
                    copy_piece<kPiece>(s_k + lane * L::kRow + i, a.kb + row * L::kRow + i);
                    copy_piece<kPiece>(s_v + lane * L::kRow + i, a.vb + row * L::kRow + i);
                }
            }
            cp_async_commit();
            scales_of<NB>(a.ks + row * NB, live, s_ks + lane * NB);
            scales_of<NB>(a.vs + row * NB, live, s_vs + lane * NB);
            cp_async_wait<0>();
            __syncwarp();
            // ---- scores ----
            float x[H];
#pragma unroll
            for (int h = 0; h < H; ++h) x[h] = 0.0f;
#pragma unroll 1
            for (int b = 0; b < NB; ++b) {
                float acc[H];
#pragma unroll
                for (int h = 0; h < H; ++h) acc[h] = 0.0f;
                uint32_t w[BITS];
#pragma unroll
                for (int i = 0; i < BITS; ++i) w[i] = reinterpret_cast<const uint32_t*>(s_k + lane * L::kRow + b * 4 * BITS)[i];
#pragma unroll
                for (int d = 0; d < 32; ++d) {
                    const int k = (BITS * d) >> 5, sh = (BITS * d) & 31;
                    const uint32_t at = sh < 7 ? w[k] << (7 - sh) : sh + BITS <= 32 ? w[k] >> (sh - 7) : __funnelshift_r(w[k], w[k + 1 < BITS ? k + 1 : k], sh - 7);
                    const float c = centroid(at);
#pragma unroll
                    for (int h = 0; h < H; h += 4) {
                        const float4 q = *reinterpret_cast<const float4*>(s_q + (b * 32 + d) * H + h);
                        acc[h] = fmaf(q.x, c, acc[h]);
                        acc[h + 1] = fmaf(q.y, c, acc[h + 1]);
                        acc[h + 2] = fmaf(q.z, c, acc[h + 2]);
                        acc[h + 3] = fmaf(q.w, c, acc[h + 3]);
                    }
                }
                const float ks = s_ks[lane * NB + b];
#pragma unroll
                for (int h = 0; h < H; ++h) x[h] = fmaf(acc[h], ks, x[h]);
            }
            // ---- softmax ----
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (!live) x[h] = -INFINITY;
                float top = x[h];
#pragma unroll
                for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
                const float to = fmaxf(m[h], top), keep = ex2(m[h] - to);
                x[h] = ex2(x[h] - to);
                m[h] = to;
                l[h] = fmaf(l[h], keep, x[h]);
#pragma unroll
                for (int b = 0; b < NB; ++b) o[h][b] *= keep;
            }
#pragma unroll
            for (int h = 0; h < H; h += 4) *reinterpret_cast<float4*>(s_p + lane * H + h) = make_float4(x[h], x[h + 1], x[h + 2], x[h + 3]);
            __syncwarp();
            // ---- values: a lane a dim ----
#pragma unroll 2
            for (int i = 0; i < last; ++i) {
                float p[H], vs[NB];
#pragma unroll
                for (int h = 0; h < H; ++h) p[h] = s_p[i * H + h];
#pragma unroll
                for (int b = 0; b < NB; ++b) vs[b] = s_vs[i * NB + b];
                const uint32_t* const codes = reinterpret_cast<const uint32_t*>(s_v + i * L::kRow);
                constexpr int kBit = BITS;
                const int word = (kBit * lane) >> 5, sh = (kBit * lane) & 31;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t w = codes[b * BITS + word];
                    if (BITS == 3) w = __funnelshift_r(w, codes[b * BITS + (sh + BITS > 32 ? word + 1 : word)], sh) << 7;
                    else w = __funnelshift_l(w, w, 7 - sh);   // (rotated: the code to bit 7)
                    const float c = centroid(w) * vs[b];
#pragma unroll
                    for (int h = 0; h < H; ++h) o[h][b] = fmaf(p[h], c, o[h][b]);
                }
            }
            __syncwarp();   // the tokens' places are free again
        }
        // ---- the segment's end ----
        const bool whole = s.whole();
        const int slot = 2 * warp + (s.begins ? 1 : 0);
        float* const to = fragment(whole ? 2 * warp + 1 : slot);
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], i);
#pragma unroll
            for (int b = 0; b < NB; ++b) to[h * D + b * 32 + lane] = o[h][b];
            if (!whole && lane == 0) {
                s_frag.m[slot][h] = m[h];
                s_frag.l[slot][h] = l[h];
            }
        }
        if (!whole && lane == 0) {
            s_frag.seg[slot] = s;
            s_frag.used[slot] = 1;
        }
        __syncwarp();
        if (whole) {
            const int quads = s.heads * (D / 4);
#pragma unroll 1
            for (int x0 = 0; x0 < quads; x0 += 32) {
                const int x = min(x0 + lane, quads - 1), hh = x / (D / 4);
                float sum = l[0];
#pragma unroll
                for (int h = 1; h < H; ++h) sum = h == hh ? l[h] : sum;
                write_quad(a.out, a.out_dtype, quad_at<NB>(a, s, x), x0 + lane < quads, reinterpret_cast<const float4*>(to)[x], sum, a.sign_mag);
            }
            __syncwarp();
        }
    }
    finish<NB>(a, s_frag, [&](int c, int x) { return reinterpret_cast<const float4*>(fragment(c))[x]; });
    write_empty<NB>(a);
}

template <int NB, int H, int BITS>
int launch_f32(const PagedArgs& a, cudaStream_t s) {
    using L = F32Plan<NB, H, BITS>;
    if (int st = allow_shared<paged_f32_kernel<NB, H, BITS>>(L::kBytes)) return st;
    paged_f32_kernel<NB, H, BITS><<<148 * L::kCtas, kWorkThreads, L::kBytes, s>>>(a);
    return check_launch(s);
}
template <int NB, int BITS>
int launch_f32_heads(const PagedArgs& a, cudaStream_t s) {
    return a.group <= 4 ? launch_f32<NB, 4, BITS>(a, s) : launch_f32<NB, 8, BITS>(a, s);
}

size_t part_bytes(int head_dim) { return sizeof(float) * (size_t)kMaxCtas * 2 * kSegHeads * (2 + 2 + head_dim); }

// cu, rows: of tqb_paged_attention_rows, or nullptr.
int attention(const tqb_paged_layer* layer, const tqb_paged_attention_params* p, const int32_t* cu, int rows, cudaStream_t s) {
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
    if (p->num_requests == 0 || (cu && rows == 0)) return TQB_OK;
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
    a.cu = cu;
    a.rows = rows;
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
    // (below 2^30 units and 2^21 heads the quotients of divide() stay below 2^21)
    if (a.vheads >= 1 << 21) return TQB_ERR_TOO_LARGE;
    auto units = [&](int shift) { return (double)a.requests * (kOpenCost + 1 + (double)((a.max_len / kRunTokens) >> shift)) * a.vheads; };
    while (units(a.unit_shift) >= 1073741824.0 && a.unit_shift < 24) ++a.unit_shift;
    if (units(a.unit_shift) >= 1073741824.0) return TQB_ERR_TOO_LARGE;
    a.q_dtype = p->q_dtype;
    a.out_dtype = p->out_dtype;
    a.qk_const = p->softmax_scale * 1.4426950408889634f;
    a.sign_mag = block_sign_magnitude();
    for (int i = 0; i < 16; ++i) a.cent[i] = cb.c[i];
    if (p->q_dtype != TQB_F32 && layer->num_pages > 0) return launch_paged_mma(a, layer->head_dim, layer->bits, s);
    switch (layer->head_dim * 10 + layer->bits) {
        case 643: return launch_f32_heads<2, 3>(a, s);
        case 644: return launch_f32_heads<2, 4>(a, s);
        case 1283: return launch_f32_heads<4, 3>(a, s);
        case 1284: return launch_f32_heads<4, 4>(a, s);
        case 2563: return launch_f32_heads<8, 3>(a, s);
        default: return launch_f32_heads<8, 4>(a, s);
    }
}

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
    return attention(layer, p, nullptr, 0, as_stream(stream));
}

int tqb_paged_attention_rows(const tqb_paged_layer* layer, const tqb_paged_attention_params* p, const int32_t* cu, int32_t num_rows,
                             tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    if (!cu) return TQB_ERR_NULL_POINTER;
    if ((uintptr_t)cu % 4 != 0) return TQB_ERR_MISALIGNED;
    if (num_rows < 0) return TQB_ERR_INVALID_ARGUMENT;
    return attention(layer, p, cu, num_rows, as_stream(stream));
}

}  // extern "C"
