// Attention of one new token of each request over the paged packed cache, 16-bit queries: the tensor-core kernel.
//
// Four warps share a segment (tqb_paged_work.cuh): warp w takes the groups of 16 tokens w, w + 4, .. of it.  The work is one
// pass over the packed bytes with the running maximum and sum of a softmax; at the measured copy bandwidth an SM
// scheduler has about 400 issue slots for 16 tokens of a KV head (4-bit, 2304 bytes), and that, not the MMAs, is what the
// layout below is about.
//
// Scores S = K~ Q~^T (mma.sync s8 x s8 -> s32, one 32-block an instruction): rows are 16 tokens, a code c enters as the byte
//   16 (c - 7.5), two logic operations for four codes; the rotated query enters as a 16-bit integer in two base-256 digits,
//   round(q~ 32639 / max |q~|), exact to 2^-16 of the head's largest component - queries come in 8 or 11 bits.  Up to four
//   heads: digits side by side in the columns (2h, 2h + 1) of one MMA; up to eight: a head a column, an MMA a digit.  The
//   block's scale multiplies the integer sum.
// Softmax: lane 4n + j has tokens n and n + 8 of head j (heads 2j, 2j + 1).  The reference m is common to the warp and only
//   raised when some score exceeds it by kShift + kLazy, which a vote finds out: no shuffles otherwise.  p = 2^(s - m), up to
//   2^(kShift + kLazy), so that f16 holds products with small weights and small scales in its normal range.
// O^T = V^T P' (mma.sync f16, K = 16 tokens): P' = p |s_v|, rounded to f16 (once for p, once for the product: 2^-11 each,
//   below the rounding of a bf16 output and within that of f16).  Up to four heads, the two columns of a head carry the
//   scales of two neighbouring blocks, one half2 product for both, and one movmatrix turns them into B fragments.
//   The codes of V enter as SUBNORMAL f16 values c 2^-23 and c 2^-19 - one mask a register, no arithmetic - and the centre 7.5
//   is taken off by starting each accumulation at -7.5 sum P', itself an MMA with constant rows.  Accumulators live for
//   32 tokens and are then added to the running output in rounded f32 additions; one long chain would add up the truncation
//   of the MMA's adder relative to 7.5 sum P'.
//   Products beyond f16 (|s_v| above 16) show as a non-finite output: the segment is then done again with smaller p.
#include "tqb_common.cuh"
#include "tqb_mma.cuh"
#include "tqb_paged.cuh"
#include "tqb_paged_work.cuh"

#include <float.h>

#include <atomic>

namespace tqb {
namespace {

constexpr int kGroupTokens = 16;
constexpr int kRing = 4;     // stages of a warp
constexpr int kStepGroups = 2;
constexpr int kInFlight = kRing - kStepGroups;
constexpr float kShift = 8.0f, kLazy = 4.0f;
constexpr float kQMax = 32639.0f;   // 127 * 256 + 127

template <int BYTES>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

// x[i]: half2 of code i of the two tokens in the halves of w, as the subnormals c 2^-23 (i even), c 2^-19 (i odd).
__device__ __forceinline__ void codes_to_subnormals(uint32_t w, uint32_t (&x)[4]) {
    const uint32_t w1 = w << 1, w7 = w >> 7;
    x[0] = w1 & 0x001e001eu;
    x[1] = w1 & 0x01e001e0u;
    x[2] = w7 & 0x001e001eu;
    x[3] = w7 & 0x01e001e0u;
}
constexpr uint32_t kCentreEven = 0x800f800fu;   // -7.5 2^-23 as a subnormal f16, twice
constexpr uint32_t kCentreOdd = 0x80f080f0u;    // -7.5 2^-19

__device__ __forceinline__ uint32_t scaled(uint32_t p, uint32_t scales) {   // p |s|, two f16 values
    return h2_as_u32(__hmul2(u32_as_h2(p), __habs2(u32_as_h2(scales))));
}

template <int NB>
struct Shape {
    static constexpr int kRow = 16 * NB;                // bytes of a token's codes
    static constexpr int kIdx = kGroupTokens * kRow;    // of a stage's K (or V) codes
    static constexpr int kSc = 2 * NB;                  // of a token's scales
    static constexpr int kStage = 2 * kIdx + 2 * kGroupTokens * kSc;   // [K codes][V codes][K scales][V scales]
    static constexpr int kWarpRing = kRing * kStage;
    // 16-byte piece c of token row t lies at piece c ^ swizzle(t): the eight rows of an ldmatrix hit different banks
    __device__ static __forceinline__ int swizzle(int t) { return NB == 2 ? (t >> 2) & 1 : NB == 4 ? (t >> 1) & 3 : t & 7; }
};

template <int NB, int HG>
struct Plan {   // CTAs of an SM, by registers and shared memory
    static constexpr int kCtas = NB == 8 ? (HG == 8 ? 2 : 3) : HG == 8 ? 4 : 5;
};

template <int NB, int HG>
__global__ void __launch_bounds__(kWorkThreads, Plan<NB, HG>::kCtas) paged_mma_kernel(const __grid_constant__ PagedArgs a) {
    using G = Shape<NB>;
    constexpr int D = NB * 32, kWarps = kWorkThreads / 32, kE = HG == 4 ? 1 : 2, kPairs = NB / 2;
    constexpr int kSets = HG == 4 ? 1 : 2;   // MMAs of a block's scores
    extern __shared__ __align__(128) unsigned char s_ring[];
    __shared__ float s_q[HG][D];
    __shared__ __align__(16) uint2 s_qfr[kSets][NB][32];
    __shared__ float s_qsc[kSegHeads];
    __shared__ float s_m[kWarps][kSegHeads], s_l[kWarps][kSegHeads];
    float* s_o = reinterpret_cast<float*>(s_ring);   // [kWarps][HG][D], when the rings are idle
    static_assert(kWarps * HG * D * 4 <= kWarps * G::kWarpRing, "outputs do not fit into the rings");

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = lane >> 2, j = lane & 3;
    const float step = 2.0f * a.cent[15] / 15.0f;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_ring) + warp * G::kWarpRing;
    // ldmatrix: lane l gives the row address of token 8 ((l >> 3) & 1) + (l & 7), block 2 pair + (l >> 4)
    const int tok = 8 * ((lane >> 3) & 1) + (lane & 7);
    const uint32_t off_k = tok * G::kRow + (((lane >> 4) ^ G::swizzle(tok)) << 4);   // ^ 32 pair
    const uint32_t off_s = 2 * G::kIdx + n * G::kSc;
    const int piece_t = lane / NB, piece_c = lane % NB;
    const uint32_t off_p = piece_t * G::kRow + ((piece_c ^ G::swizzle(piece_t)) << 4);
    const uint32_t off_ps = 2 * G::kIdx + lane * G::kSc;   // K scales of tokens 0..15, V scales behind them
    const int mask = (1 << a.page_shift) - 1;

    WorkLine line(a);
    write_empty<NB>(a);
    while (line.more()) {
        const Segment s = line.next();
        __syncthreads();   // the last segment's end has read the shared arrays

        // ---- queries: rotated, scaled to integers, cut into digits ----
        {
            const float inv_sqrt = 1.0f / sqrtf((float)kBlock), sg = block_sign(lane, a.sign_mag);
#pragma unroll 4
            for (int u = warp; u < HG * NB; u += kWarps) {
                const int hh = u / NB, b = u - hh * NB;
                float v = hh < s.heads ? load_as_f32(a.q, a.q_dtype, (size_t)s.req * a.q_stride + (size_t)(s.head0 + hh) * D + b * 32 + lane) : 0.0f;
                s_q[hh][b * 32 + lane] = wht32_across(v, lane) * inv_sqrt * sg;
            }
        }
        // ---- the segment's groups of this warp ----
        const int first = s.t0 + warp * kGroupTokens, last = s.t1 - 1;
        const int groups = first < s.t1 ? (s.t1 - first + kTile - 1) / kTile : 0;
        const int steps = (groups + kStepGroups - 1) / kStepGroups * kStepGroups;
        const int32_t* table = a.table + (size_t)s.req * a.table_stride;
        auto page_of = [&](int i) { return table[min(first + i * kTile, last) >> a.page_shift]; };
        __syncthreads();
        for (int hh = warp; hh < HG; hh += kWarps) {
            uint32_t top = 0;   // of the bits, so that NaN is above infinity
#pragma unroll
            for (int i = 0; i < NB; ++i) top = max(top, __float_as_uint(s_q[hh][lane + 32 * i]) & 0x7fffffffu);
            top = __reduce_max_sync(0xffffffffu, top);
            const float m = __uint_as_float(top);
            if (lane == 0) s_qsc[hh] = m <= FLT_MAX ? m : __uint_as_float(0x7fc00000u);   // not finite: every score is NaN
        }
        __syncthreads();
        for (int b = warp; b < NB; b += kWarps) {
            const int hh = HG == 4 ? n >> 1 : n;
            const float m = s_qsc[hh], inv = m > 0.0f && m <= FLT_MAX ? kQMax / m : 0.0f;
            uint32_t d0[2] = {0u, 0u}, d1[2] = {0u, 0u};   // [dims 8j + even | 8j + odd]
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = s_q[hh][32 * b + 8 * j + 2 * i + half];
                    const int v = inv > 0.0f ? __float2int_rn(x * inv) : 0;
                    const int lo = (int)(signed char)(v & 0xff);
                    d0[half] |= (uint32_t)(lo & 0xff) << (8 * i);
                    d1[half] |= (uint32_t)(((v - lo) >> 8) & 0xff) << (8 * i);
                }
            if (HG == 4) {
                s_qfr[0][b][lane] = (n & 1) ? make_uint2(d0[0], d0[1]) : make_uint2(d1[0], d1[1]);
            } else {
                s_qfr[0][b][lane] = make_uint2(d1[0], d1[1]);
                s_qfr[kSets - 1][b][lane] = make_uint2(d0[0], d0[1]);
            }
        }
        float qsc[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) qsc[e] = s_qsc[HG == 4 ? j : 2 * j + e] * (a.qk_const * step / (kQMax * 16.0f));
        __syncthreads();
        const uint32_t qfr = (uint32_t)__cvta_generic_to_shared(&s_qfr[0][0][lane]);

        float shift = kShift;
        float m_ref[kE], l_run[kE];
        float o[NB][2][HG == 4 ? 2 : 4];
        for (;;) {
            float thr[kE];
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                m_ref[e] = thr[e] = kNoScore;
                l_run[e] = 0.0f;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < (HG == 4 ? 2 : 4); ++i) o[b][m][i] = 0.0f;
            int page_now = page_of(lane), page_next = page_of(32 + lane);
            uint32_t bad = 0;   // groups in flight whose page does not exist: bit (group & 31)
            uint32_t st_fill = ring, st = ring;
            auto fill = [&](int i) {
                if ((i & 31) == 0 && i > 0) {
                    page_now = page_next;
                    page_next = page_of(i + 32 + lane);
                }
                int page = __shfl_sync(0xffffffffu, page_now, i & 31);
                const uint32_t bit = 1u << (i & 31);
                bad &= ~bit;
                if ((unsigned)page >= (unsigned)a.num_pages) {
                    bad |= bit;
                    page = 0;
                }
                if (i < steps) {
                    const int gs = first + i * kTile;
                    const uint32_t base = ((uint32_t)page * a.hkv + s.kvh) << a.page_shift;
                    const uint16_t* scb = (lane < 16 ? a.ks : a.vs);
                    if (gs + kGroupTokens <= s.t1) {
                        const uint32_t row = base + (gs & mask);
                        const uint8_t* k = a.kb + (size_t)row * G::kRow + lane * 16;
                        const uint8_t* v = a.vb + (size_t)row * G::kRow + lane * 16;
#pragma unroll
                        for (int p = 0; p < G::kRow / 32; ++p) {
                            const uint32_t d = st_fill + (NB == 8 && (p & 1) ? off_p ^ 64 : off_p) + p * 512;
                            cp_async16(d, k + p * 512);
                            cp_async16(d + G::kIdx, v + p * 512);
                        }
                        cp_async_small<G::kSc>(st_fill + off_ps, scb + (size_t)(row + (lane & 15)) * NB);
                    } else {   // rows behind the segment's last token read that one; they are masked
#pragma unroll
                        for (int p = 0; p < G::kRow / 32; ++p) {
                            const uint32_t row = base + (min(gs + piece_t + p * (32 / NB), last) & mask);
                            const size_t at = (size_t)row * G::kRow + piece_c * 16;
                            const uint32_t d = st_fill + (NB == 8 && (p & 1) ? off_p ^ 64 : off_p) + p * 512;
                            cp_async16(d, a.kb + at);
                            cp_async16(d + G::kIdx, a.vb + at);
                        }
                        const uint32_t row = base + (min(gs + (lane & 15), last) & mask);
                        cp_async_small<G::kSc>(st_fill + off_ps, scb + (size_t)row * NB);
                    }
                }
                cp_async_commit();
                st_fill = st_fill + G::kStage == ring + G::kWarpRing ? ring : st_fill + G::kStage;
            };
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) fill(i);
            for (int it = 0; it < steps; it += kStepGroups) {
#pragma unroll
                for (int u = 0; u < kStepGroups; ++u) fill(it + kInFlight + u);
                cp_async_wait<kInFlight>();
                __syncwarp();
                uint32_t stu[kStepGroups];
#pragma unroll
                for (int u = 0; u < kStepGroups; ++u) {
                    stu[u] = st;
                    st = st + G::kStage == ring + G::kWarpRing ? ring : st + G::kStage;
                }
                // ---- scores ----
                float sc[kStepGroups][2][kE];
                static_for<0, kStepGroups>([&](auto u_) {
                    constexpr int u = decltype(u_)::value;
                    float acc[2][kE];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < kE; ++e) acc[t][e] = 0.0f;
                    static_for<0, kPairs>([&](auto p_) {
                        constexpr int p = decltype(p_)::value;
                        uint32_t kw[4];
                        ldsm4_o<0>(stu[u] + (off_k ^ (32 * p)), kw);
                        const uint32_t sa = lds32_o<4 * p>(stu[u] + off_s), sb = lds32_o<4 * p + 8 * G::kSc>(stu[u] + off_s);
                        static_for<0, 2>([&](auto i_) {
                            constexpr int i = decltype(i_)::value, b = 2 * p + i;
                            const float ka = fabsf(i ? __high2float(u32_as_h2(sa)) : __low2float(u32_as_h2(sa)));
                            const float kb = fabsf(i ? __high2float(u32_as_h2(sb)) : __low2float(u32_as_h2(sb)));
                            // c ^ 8 is the two's complement of c - 8; at the top of a byte with bit 3 set below it: 16 (c - 7.5)
                            const uint32_t u0 = kw[2 * i] ^ 0x88888888u, u1 = kw[2 * i + 1] ^ 0x88888888u;
                            const uint32_t a0 = lop3_and_or(u0 << 4, 0xF0F0F0F0u, 0x08080808u), a2 = lop3_and_or(u0, 0xF0F0F0F0u, 0x08080808u);
                            const uint32_t a1 = lop3_and_or(u1 << 4, 0xF0F0F0F0u, 0x08080808u), a3 = lop3_and_or(u1, 0xF0F0F0F0u, 0x08080808u);
                            const uint2 qa = lds64_o<b * 256>(qfr);
                            int hi[4];
                            imma16832(hi, a0, a1, a2, a3, qa.x, qa.y);
                            if (HG == 4) {
                                acc[0][0] = fmaf(ka, (float)(hi[0] * 256 + hi[1]), acc[0][0]);
                                acc[1][0] = fmaf(kb, (float)(hi[2] * 256 + hi[3]), acc[1][0]);
                            } else {
                                const uint2 qb = lds64_o<(NB + b) * 256>(qfr);
                                int lo[4];
                                imma16832(lo, a0, a1, a2, a3, qb.x, qb.y);
#pragma unroll
                                for (int e = 0; e < kE; ++e) {
                                    acc[0][e] = fmaf(ka, (float)(hi[e] * 256 + lo[e]), acc[0][e]);
                                    acc[1][e] = fmaf(kb, (float)(hi[2 + e] * 256 + lo[2 + e]), acc[1][e]);
                                }
                            }
                        });
                    });
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < kE; ++e) sc[u][t][e] = acc[t][e] * qsc[e];
                    const int gs = first + (it + u) * kTile;
                    const bool none = (bad >> ((it + u) & 31)) & 1u;
                    if (none || gs + kGroupTokens > s.t1) {
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            if (none || gs + n + 8 * t >= s.t1) {
#pragma unroll
                                for (int e = 0; e < kE; ++e) sc[u][t][e] = -INFINITY;
                            }
                    }
                });
                // ---- softmax ----
                bool over = false;
                float top[kE];
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    top[e] = fmaxf(fmaxf(sc[0][0][e], sc[0][1][e]), fmaxf(sc[1][0][e], sc[1][1][e]));
                    over |= top[e] > thr[e];
                }
                if (__any_sync(0xffffffffu, over)) {
                    float keep[kE];
#pragma unroll
                    for (int e = 0; e < kE; ++e) {
                        float mx = top[e];
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float m_new = mx > thr[e] ? mx - shift : m_ref[e];
                        keep[e] = ex2(m_ref[e] - m_new);
                        m_ref[e] = m_new;
                        thr[e] = m_new + (shift + kLazy);
                        l_run[e] *= keep[e];
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            if (HG == 4) {
                                o[b][m][0] *= keep[0];
                                o[b][m][1] *= keep[0];
                            } else {
#pragma unroll
                                for (int i = 0; i < (HG == 4 ? 2 : 4); ++i) o[b][m][i] *= keep[i % kE];
                            }
                        }
                }
                // ---- P' = p |s_v| as B fragments ----
                uint32_t pq[kStepGroups][HG == 4 ? kPairs : NB][2];   // [octet]
                static_for<0, kStepGroups>([&](auto u_) {
                    constexpr int u = decltype(u_)::value;
                    static_for<0, 2>([&](auto t_) {
                        constexpr int t = decltype(t_)::value;
                        float p[kE];
#pragma unroll
                        for (int e = 0; e < kE; ++e) {
                            p[e] = ex2(sc[u][t][e] - m_ref[e]);
                            l_run[e] += p[e];
                        }
                        const uint32_t ph = h2_as_u32(__floats2half2_rn(p[0], p[kE - 1]));
                        static_for<0, kPairs>([&](auto p_) {
                            constexpr int pr = decltype(p_)::value;
                            const uint32_t sv = lds32_o<16 * G::kSc + 8 * t * G::kSc + 4 * pr>(stu[u] + off_s);
                            if (HG == 4) {   // columns 2j, 2j + 1: head j with the scales of blocks 2 pr, 2 pr + 1
                                pq[u][pr][t] = movmatrix_trans(scaled(ph, sv));
                            } else {         // columns 2j, 2j + 1: heads 2j, 2j + 1
                                pq[u][2 * pr][t] = movmatrix_trans(scaled(ph, __byte_perm(sv, sv, 0x1010)));
                                pq[u][2 * pr + (HG == 4 ? 0 : 1)][t] = movmatrix_trans(scaled(ph, __byte_perm(sv, sv, 0x3232)));
                            }
                        });
                    });
                });
                // ---- O^T += V^T P' ----
                static_for<0, kPairs>([&](auto p_) {
                    constexpr int pr = decltype(p_)::value;
                    uint32_t vw[kStepGroups][4];
#pragma unroll
                    for (int u = 0; u < kStepGroups; ++u) ldsm4t_o<G::kIdx>(stu[u] + (off_k ^ (32 * pr)), vw[u]);
                    float centre[4];
                    if (HG == 4) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) centre[i] = 0.0f;
#pragma unroll
                        for (int u = 0; u < kStepGroups; ++u)
                            mma16816(centre, kCentreEven, kCentreOdd, kCentreEven, kCentreOdd, pq[u][pr][0], pq[u][pr][1]);
                    }
                    static_for<0, 2>([&](auto i_) {
                        constexpr int i = decltype(i_)::value, b = 2 * pr + i, f = HG == 4 ? pr : b;
                        if (HG == 8) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) centre[k] = 0.0f;
#pragma unroll
                            for (int u = 0; u < kStepGroups; ++u)
                                mma16816(centre, kCentreEven, kCentreOdd, kCentreEven, kCentreOdd, pq[u][f][0], pq[u][f][1]);
                        }
                        float acc[2][4];
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int k = 0; k < 4; ++k) acc[m][k] = centre[k];
#pragma unroll
                        for (int u = 0; u < kStepGroups; ++u) {
                            uint32_t xa[4], xb[4];   // tokens 2j, 2j + 1 and 2j + 8, 2j + 9: codes 4n .. 4n + 3 of the block
                            codes_to_subnormals(vw[u][2 * i], xa);
                            codes_to_subnormals(vw[u][2 * i + 1], xb);
#pragma unroll
                            for (int m = 0; m < 2; ++m)
                                mma16816(acc[m], xa[2 * m], xa[2 * m + 1], xb[2 * m], xb[2 * m + 1], pq[u][f][0], pq[u][f][1]);
                        }
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            if (HG == 4) {
                                o[b][m][0] += acc[m][i];
                                o[b][m][1] += acc[m][2 + i];
                            } else {
#pragma unroll
                                for (int k = 0; k < (HG == 4 ? 2 : 4); ++k) o[b][m][k] += acc[m][k];
                            }
                        }
                    });
                });
                __syncwarp();   // the stages may be filled again
            }
            cp_async_wait<0>();
            bool finite = true;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < (HG == 4 ? 2 : 4); ++i) finite = finite && fabsf(o[b][m][i]) <= FLT_MAX;
            // (also: all rings are idle now)
            if (!__syncthreads_or(finite ? 0 : 1) || shift < 0.0f) break;
            shift -= 6.0f;   // 8, 2, -4: p |s_v| is at most 65504 with the last
        }

        // ---- the warps' parts ----
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            float l = l_run[e];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            if (n == 0) {
                s_m[warp][HG == 4 ? j : 2 * j + e] = m_ref[e];
                s_l[warp][HG == 4 ? j : 2 * j + e] = l;
            }
        }
        const float even = step * 8388608.0f, odd = step * 524288.0f;   // 2^23, 2^19
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int d = 32 * b + 4 * n + 2 * m;   // rows n / n + 8 of the MMA are dims d / d + 1
                if (HG == 4) {
                    *reinterpret_cast<float2*>(s_o + (warp * HG + j) * D + d) = make_float2(o[b][m][0] * even, o[b][m][1] * odd);
                } else {
#pragma unroll
                    for (int e = 0; e < kE; ++e)
                        *reinterpret_cast<float2*>(s_o + (warp * HG + 2 * j + e) * D + d) = make_float2(o[b][m][e] * even, o[b][m][(HG == 4 ? 0 : 2) + e] * odd);
                }
            }
        __syncthreads();
        finish_segment<NB>(a, s, s_m, s_l, [&](int w, int h, int d) { return s_o[(w * HG + h) * D + d]; });
    }
}

template <int NB, int HG>
int launch(const PagedArgs& a, cudaStream_t s) {
    const int dyn = (kWorkThreads / 32) * Shape<NB>::kWarpRing;
    // more than 48 KB of dynamic shared memory is a property of the kernel on a device: set once for each
    static std::atomic<unsigned long long> configured{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
    if (dev < 0 || !((configured.load(std::memory_order_acquire) >> dev) & 1ull)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_mma_kernel<NB, HG>, cudaFuncAttributeMaxDynamicSharedMemorySize, dyn);
        if (e != cudaSuccess) {
            set_cuda_error(e);
            return TQB_ERR_CUDA;
        }
        if (dev >= 0) configured.fetch_or(1ull << dev, std::memory_order_release);
    }
    paged_mma_kernel<NB, HG><<<148 * Plan<NB, HG>::kCtas, kWorkThreads, dyn, s>>>(a);
    return check_launch(s);
}

}  // namespace

int launch_paged_mma(const PagedArgs& a, int head_dim, cudaStream_t s) {
    const bool narrow = a.group <= 4;
    if (head_dim == 64) return narrow ? launch<2, 4>(a, s) : launch<2, 8>(a, s);
    if (head_dim == 128) return narrow ? launch<4, 4>(a, s) : launch<4, 8>(a, s);
    return narrow ? launch<8, 4>(a, s) : launch<8, 8>(a, s);
}

}  // namespace tqb
