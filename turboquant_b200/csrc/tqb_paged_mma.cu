// Attention of one new token of each request over the paged packed cache, 16-bit queries: the tensor-core kernel.
//
// Every warp takes its segments (tqb_paged_work.cuh) by itself, two groups of 16 tokens a step, the next two in flight.  The work
// is one pass over the packed bytes with the running maximum and sum of a softmax; at the measured copy bandwidth an SM
// scheduler has about 400 issue slots for 16 tokens of a KV head (4-bit, head_dim 128: 2304 bytes), and that, not the MMAs, is
// what the layout below is about.
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

__device__ __forceinline__ uint32_t product(uint32_t a, uint32_t b) { return h2_as_u32(__hmul2(u32_as_h2(a), u32_as_h2(b))); }

template <int NB>
struct Shape {
    static constexpr int kRow = 16 * NB;                // bytes of a token's codes
    static constexpr int kIdx = kGroupTokens * kRow;    // of a stage's K (or V) codes
    static constexpr int kSc = 2 * NB;                  // of a token's scales
    static constexpr int kStage = 2 * kIdx + 2 * kGroupTokens * kSc;   // [K codes][V codes][K scales][V scales]
    static constexpr int kWarpRing = kRing * kStage;      // of a warp
    // 16-byte piece c of token row t lies at piece c ^ swizzle(t): the eight rows of an ldmatrix hit different banks
    __device__ static __forceinline__ int swizzle(int t) { return NB == 2 ? (t >> 2) & 1 : NB == 4 ? (t >> 1) & 3 : t & 7; }
};

template <int NB, int HG>
struct Plan {
    using G = Shape<NB>;
    static constexpr int kSets = HG == 4 ? 1 : 2;                 // MMAs of a block's scores
    static constexpr int kFragment = HG * NB * 32 * 4;            // outputs of a segment
    static constexpr int kDigits = kSets * NB * 32 * 8;           // the queries' MMA fragments
    static constexpr int kWarpBytes = G::kWarpRing + kFragment + kDigits;   // [ring][fragment that began before][digits]
    static constexpr int kBytes = kWorkWarps * kWarpBytes;
    // CTAs of an SM: by shared memory, and so that registers do not spill
    static constexpr int kByShared = 227 * 1024 / (kBytes + 4096), kByRegs = NB == 8 ? (HG == 8 ? 2 : 3) : HG == 8 ? 4 : NB == 2 ? 5 : 4;
    static constexpr int kCtas = kByShared < kByRegs ? kByShared : kByRegs;
};

template <int NB, int HG>
__global__ void __launch_bounds__(kWorkThreads, Plan<NB, HG>::kCtas) paged_mma_kernel(const __grid_constant__ PagedArgs a) {
    using G = Shape<NB>;
    using L = Plan<NB, HG>;
    constexpr int D = NB * 32, kE = HG == 4 ? 1 : 2, kPairs = NB / 2;
    constexpr int kO = HG == 4 ? 2 : 4;               // outputs that a lane holds of an MMA tile
    extern __shared__ __align__(128) unsigned char s_dyn[];
    __shared__ Fragments s_frag;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, j = lane & 3;
    const float step = 2.0f * a.cent[15] / 15.0f;
    unsigned char* const s_warp = s_dyn + warp * L::kWarpBytes;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_warp);
    unsigned char* const s_digits = s_warp + G::kWarpRing + L::kFragment;
    const uint32_t digits = (uint32_t)__cvta_generic_to_shared(s_digits) + lane * 8;
    const uint32_t halves = 2 * ring + kInFlight * G::kStage;   // (one half's address) + (the other's)
    static_assert(kRing == 2 * kInFlight && kStepGroups == kInFlight, "the ring has two halves of a step each");
    static_assert(L::kFragment <= G::kWarpRing, "a segment's outputs do not fit into the ring");
    // a fragment's outputs [HG][D]: that of the warp's last segment lies in its idle ring
    auto fragment = [&](int slot) { return reinterpret_cast<float*>(s_dyn + (slot >> 1) * L::kWarpBytes + ((slot & 1) ? 0 : G::kWarpRing)); };
    // ldmatrix: lane l gives the row address of token 8 ((l >> 3) & 1) + (l & 7), block 2 pair + (l >> 4)
    const int tok = 8 * ((lane >> 3) & 1) + (lane & 7);
    const uint32_t off_k = tok * G::kRow + (((lane >> 4) ^ G::swizzle(tok)) << 4);   // ^ 32 pair
    const uint32_t off_s = 2 * G::kIdx + n * G::kSc;
    const int piece_t = lane / NB, piece_c = lane % NB;
    const uint32_t off_p = piece_t * G::kRow + ((piece_c ^ G::swizzle(piece_t)) << 4);
    const uint32_t off_ps = 2 * G::kIdx + lane * G::kSc;   // K scales of tokens 0..15, V scales behind them
    const int mask = (1 << a.page_shift) - 1;

    if (threadIdx.x < 2 * kWorkWarps) s_frag.used[threadIdx.x] = 0;
    WorkLine line(a);   // (its barriers stand before the first use of what is set above)

    // ---- copies of a segment's groups, one behind the other ----
    Segment s{};
    int to_copy;                              // first token of the group that is copied next
    int page_now, page_next;                  // pages 32 k + lane of the segment, for this k and the next
    bool some_bad = false;                    // some page does not exist (of those looked at so far)
    const uint8_t *kp, *vp;
    const uint16_t* sp;
    auto page_at = [&](int i) {               // of the segment's i-th page
        const int page = a.table[s.req * a.table_stride + min((s.t0 >> a.page_shift) + i, (s.t1 - 1) >> a.page_shift)];
        const bool bad = (unsigned)page >= (unsigned)a.num_pages;
        some_bad |= __any_sync(0xffffffffu, bad) != 0;
        return bad ? 0 : page;
    };
    auto open = [&]() {
        some_bad = false;
        to_copy = s.t0;
        page_now = page_at(lane);
        page_next = (s.t1 - 1) >> a.page_shift >= (s.t0 >> a.page_shift) + 32 ? page_at(32 + lane) : 0;
    };
    auto fill = [&](uint32_t st) {
        if (to_copy < s.t1) {
            if ((to_copy & mask) == 0 || to_copy == s.t0) {
                const int i = (to_copy >> a.page_shift) - (s.t0 >> a.page_shift);
                if (i > 0 && (i & 31) == 0) {
                    page_now = page_next;
                    page_next = page_at(i + 32 + lane);
                }
                const int page = __shfl_sync(0xffffffffu, page_now, i & 31);
                const uint32_t row = (((uint32_t)page * a.hkv + s.kvh) << a.page_shift) + (to_copy & mask);
                kp = a.kb + (size_t)row * G::kRow + lane * 16;
                vp = a.vb + (size_t)row * G::kRow + lane * 16;
                sp = (lane < 16 ? a.ks : a.vs) + (size_t)(row + (lane & 15)) * NB;
            }
            // whole groups, also where the request ends inside: the page has the room
#pragma unroll
            for (int p = 0; p < G::kRow / 32; ++p) {
                const uint32_t d = st + (NB == 8 && (p & 1) ? off_p ^ 64 : off_p) + p * 512;
                cp_async16(d, kp + p * 512);
                cp_async16(d + G::kIdx, vp + p * 512);
            }
            cp_async_small<G::kSc>(st + off_ps, sp);
            kp += G::kIdx;
            vp += G::kIdx;
            sp += kGroupTokens * NB;
        }
        cp_async_commit();
        to_copy += kGroupTokens;
    };

    while (line.next(s)) {
        // ---- queries: rotated, scaled to integers, cut into digits ----
        float qsc[kE];
        {
            constexpr int kAtOnce = HG * NB <= 32 ? HG : 4;   // heads
            const float inv_sqrt = 1.0f / sqrtf((float)kBlock), sg = block_sign(lane, a.sign_mag);
            const size_t q0 = (size_t)s.req * a.q_stride + (size_t)s.head0 * D + lane;
#pragma unroll
            for (int e = 0; e < kE; ++e) qsc[e] = 0.0f;
            // Byte i of k-slots 4j' + i of fragment (b, 4n' + j') is dim 32 b + 8 j' + 2 i (first word) or one above it (second), of
            // column n': this lane's dim has j' = lane / 8, i = lane / 2 % 4, word lane % 2
            unsigned char* const at = s_digits + (lane >> 3) * 8 + (lane & 1) * 4 + ((lane >> 1) & 3);
#pragma unroll
            for (int h0 = 0; h0 < HG; h0 += kAtOnce) {
                float v[kAtOnce][NB];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                    for (int b = 0; b < NB; ++b) v[i][b] = h0 + i < s.heads ? load_as_f32(a.q, a.q_dtype, q0 + (h0 + i) * D + b * 32) : 0.0f;
                if (h0 == 0) {   // (behind the queries' loads)
                    open();
#pragma unroll
                    for (int i = 0; i < kInFlight; ++i) fill(ring + i * G::kStage);
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const int h = h0 + i;
                    uint32_t top = 0;   // of the bits, so that NaN is above infinity
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        v[i][b] = wht32_across(v[i][b], lane) * inv_sqrt * sg;
                        top = max(top, __float_as_uint(v[i][b]) & 0x7fffffffu);
                    }
                    float m = __uint_as_float(__reduce_max_sync(0xffffffffu, top));
                    if (!(m <= FLT_MAX)) m = __uint_as_float(0x7fc00000u);   // not finite: every score is NaN
                    const float inv = m > 0.0f ? kQMax / m : 0.0f;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        // (inv is infinite where the largest component is below 1e-34)
                        const int x = inv <= FLT_MAX ? __float2int_rn(v[i][b] * inv) : 0;
                        const int lo = (int)(signed char)(x & 0xff), hi = (x - lo) >> 8;
                        if (HG == 4) {
                            at[b * 256 + (2 * h) * 32] = (unsigned char)hi;
                            at[b * 256 + (2 * h + 1) * 32] = (unsigned char)lo;
                        } else {
                            at[b * 256 + h * 32] = (unsigned char)hi;
                            at[(NB + b) * 256 + h * 32] = (unsigned char)lo;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < kE; ++e)
                        if (h == (HG == 4 ? j : 2 * j + e)) qsc[e] = m * (a.qk_const * step / (kQMax * 16.0f));
                }
            }
            __syncwarp();
        }

        float shift = kShift;
        float m_ref[kE], l_run[kE];
        float o[NB][2][kO];
        for (;;) {
#pragma unroll
            for (int e = 0; e < kE; ++e) {
                m_ref[e] = kNoScore;
                l_run[e] = 0.0f;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < kO; ++i) o[b][m][i] = 0.0f;
            uint32_t st = ring;
            for (int t0 = s.t0; t0 < s.t1; t0 += kStepGroups * kGroupTokens) {
                const uint32_t st_other = halves - st;
#pragma unroll
                for (int u = 0; u < kStepGroups; ++u) fill(st_other + u * G::kStage);
                cp_async_wait<kInFlight>();
                __syncwarp();
                // ---- scores ----
                float raw[kStepGroups][2][kE];
                static_for<0, kStepGroups>([&](auto u_) {
                    constexpr int u = decltype(u_)::value;
                    const uint32_t stu = st + u * G::kStage;
                    float acc[2][kE];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < kE; ++e) acc[t][e] = 0.0f;
                    static_for<0, kPairs>([&](auto p_) {
                        constexpr int p = decltype(p_)::value;
                        uint32_t kw[4];
                        ldsm4_o<0>(stu + (off_k ^ (32 * p)), kw);
                        const uint32_t sa = lds32_o<4 * p>(stu + off_s) & 0x7fff7fffu, sb = lds32_o<4 * p + 8 * G::kSc>(stu + off_s) & 0x7fff7fffu;
                        static_for<0, 2>([&](auto i_) {
                            constexpr int i = decltype(i_)::value, b = 2 * p + i;
                            const float ka = i ? __high2float(u32_as_h2(sa)) : __low2float(u32_as_h2(sa));
                            const float kc = i ? __high2float(u32_as_h2(sb)) : __low2float(u32_as_h2(sb));
                            // c ^ 8 is the two's complement of c - 8; at the top of a byte with bit 3 set below it: 16 (c - 7.5)
                            const uint32_t u0 = kw[2 * i], u1 = kw[2 * i + 1];
                            const uint32_t a0 = lop3_xor_select(u0 << 4, 0xF0F0F0F0u, 0x88888888u), a2 = lop3_xor_select(u0, 0xF0F0F0F0u, 0x88888888u);
                            const uint32_t a1 = lop3_xor_select(u1 << 4, 0xF0F0F0F0u, 0x88888888u), a3 = lop3_xor_select(u1, 0xF0F0F0F0u, 0x88888888u);
                            const uint2 qa = lds64_o<b * 256>(digits);
                            int hi[4];
                            imma16832(hi, a0, a1, a2, a3, qa.x, qa.y);
                            if constexpr (HG == 4) {
                                acc[0][0] = fmaf(ka, (float)(hi[0] * 256 + hi[1]), acc[0][0]);
                                acc[1][0] = fmaf(kc, (float)(hi[2] * 256 + hi[3]), acc[1][0]);
                            } else {
                                const uint2 qb = lds64_o<(NB + b) * 256>(digits);
                                int lo[4];
                                imma16832(lo, a0, a1, a2, a3, qb.x, qb.y);
#pragma unroll
                                for (int e = 0; e < kE; ++e) {
                                    acc[0][e] = fmaf(ka, (float)(hi[e] * 256 + lo[e]), acc[0][e]);
                                    acc[1][e] = fmaf(kc, (float)(hi[2 + e] * 256 + lo[2 + e]), acc[1][e]);
                                }
                            }
                        });
                    });
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < kE; ++e) raw[u][t][e] = acc[t][e];
                });
                // Tokens behind the segment's end and those of pages that do not exist: no score, and no scale of theirs meets a
                // zero weight (it may be infinite or NaN).
                bool out[kStepGroups][2];
                uint32_t sv_mask[kStepGroups][2];
#pragma unroll
                for (int u = 0; u < kStepGroups; ++u)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        out[u][t] = false;
                        sv_mask[u][t] = 0x7fff7fffu;
                    }
                if (some_bad || t0 + kStepGroups * kGroupTokens > s.t1) {
#pragma unroll
                    for (int u = 0; u < kStepGroups; ++u) {
                        const int gs = t0 + u * kGroupTokens;
                        const bool none = some_bad && (unsigned)a.table[s.req * a.table_stride + (min(gs, s.t1 - 1) >> a.page_shift)] >= (unsigned)a.num_pages;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            if (none || gs + n + 8 * t >= s.t1) {
                                out[u][t] = true;
                                sv_mask[u][t] = 0u;
                            }
                    }
                }
                // ---- softmax ----
                float x[kStepGroups][2][kE];
                bool over = false;
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    float top = -INFINITY;
#pragma unroll
                    for (int u = 0; u < kStepGroups; ++u)
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            x[u][t][e] = out[u][t] ? -INFINITY : fmaf(raw[u][t][e], qsc[e], -m_ref[e]);
                            top = fmaxf(top, x[u][t][e]);
                        }
                    over |= top > shift + kLazy;
                }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int e = 0; e < kE; ++e) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int u = 0; u < kStepGroups; ++u)
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                if (!out[u][t]) mx = fmaxf(mx, raw[u][t][e] * qsc[e]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float m_new = fmaxf(m_ref[e], mx - shift), keep = ex2(m_ref[e] - m_new);
                        m_ref[e] = m_new;
                        l_run[e] *= keep;
#pragma unroll
                        for (int u = 0; u < kStepGroups; ++u)
#pragma unroll
                            for (int t = 0; t < 2; ++t) x[u][t][e] = out[u][t] ? -INFINITY : fmaf(raw[u][t][e], qsc[e], -m_new);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int m = 0; m < 2; ++m)
#pragma unroll
                                for (int i = 0; i < kO; ++i)
                                    if (HG == 4 || i % 2 == e) o[b][m][i] *= keep;
                    }
                }
                // ---- P' = p |s_v| as B fragments ----
                uint32_t pq[kStepGroups][HG == 4 ? kPairs : NB][2];   // [octet]
                static_for<0, kStepGroups>([&](auto u_) {
                    constexpr int u = decltype(u_)::value;
                    const uint32_t stu = st + u * G::kStage;
                    static_for<0, 2>([&](auto t_) {
                        constexpr int t = decltype(t_)::value;
                        float p[kE];
#pragma unroll
                        for (int e = 0; e < kE; ++e) {
                            p[e] = ex2(x[u][t][e]);
                            l_run[e] += p[e];
                        }
                        const uint32_t ph = h2_as_u32(__floats2half2_rn(p[0], p[kE - 1]));
                        static_for<0, kPairs>([&](auto p_) {
                            constexpr int pr = decltype(p_)::value;
                            const uint32_t sv = lds32_o<16 * G::kSc + 8 * t * G::kSc + 4 * pr>(stu + off_s) & sv_mask[u][t];
                            if constexpr (HG == 4) {   // columns 2j, 2j + 1: head j with the scales of blocks 2 pr, 2 pr + 1
                                pq[u][pr][t] = movmatrix_trans(product(ph, sv));
                            } else {                   // columns 2j, 2j + 1: heads 2j, 2j + 1
                                pq[u][2 * pr][t] = movmatrix_trans(product(ph, __byte_perm(sv, sv, 0x1010)));
                                pq[u][2 * pr + 1][t] = movmatrix_trans(product(ph, __byte_perm(sv, sv, 0x3232)));
                            }
                        });
                    });
                });
                // ---- O^T += V^T P' ----
                const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                static_for<0, kPairs>([&](auto p_) {
                    constexpr int pr = decltype(p_)::value;
                    uint32_t vw[kStepGroups][4];
#pragma unroll
                    for (int u = 0; u < kStepGroups; ++u) ldsm4t_o<G::kIdx>(st + u * G::kStage + (off_k ^ (32 * pr)), vw[u]);
                    float centre[4];
                    static_for<0, 2>([&](auto i_) {
                        constexpr int i = decltype(i_)::value, b = 2 * pr + i, f = HG == 4 ? pr : b;
                        if (HG == 8 || i == 0) {
                            mma16816_from(centre, zero, kCentreEven, kCentreOdd, kCentreEven, kCentreOdd, pq[0][f][0], pq[0][f][1]);
#pragma unroll
                            for (int u = 1; u < kStepGroups; ++u)
                                mma16816(centre, kCentreEven, kCentreOdd, kCentreEven, kCentreOdd, pq[u][f][0], pq[u][f][1]);
                        }
                        float acc[2][4];
#pragma unroll
                        for (int u = 0; u < kStepGroups; ++u) {
                            uint32_t xa[4], xb[4];   // tokens 2j, 2j + 1 and 2j + 8, 2j + 9: codes 4n .. 4n + 3 of the block
                            codes_to_subnormals(vw[u][2 * i], xa);
                            codes_to_subnormals(vw[u][2 * i + 1], xb);
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                if (u == 0) mma16816_from(acc[m], centre, xa[2 * m], xa[2 * m + 1], xb[2 * m], xb[2 * m + 1], pq[u][f][0], pq[u][f][1]);
                                else mma16816(acc[m], xa[2 * m], xa[2 * m + 1], xb[2 * m], xb[2 * m + 1], pq[u][f][0], pq[u][f][1]);
                            }
                        }
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int k = 0; k < kO; ++k) o[b][m][k] += HG == 4 ? acc[m][2 * k + i] : acc[m][k];
                    });
                });
                __syncwarp();   // the stages may be filled again
                st = st_other;
            }
            cp_async_wait<0>();
            __syncwarp();
            bool finite = true;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < kO; ++i) finite = finite && fabsf(o[b][m][i]) <= FLT_MAX;
            if (__all_sync(0xffffffffu, finite) || shift < 0.0f) break;
            shift -= 6.0f;   // 8, 2, -4: with the last, p |s_v| is at most 65504
            open();
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) fill(ring + i * G::kStage);
        }

        // ---- the segment's end ----
        const bool whole = s.whole();
        const int slot = 2 * warp + (s.begins ? 1 : 0);
        float* const to = fragment(slot);
        const float even = step * 8388608.0f, odd = step * 524288.0f;   // 2^23, 2^19
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int d = 32 * b + 4 * n + 2 * m;   // rows n / n + 8 of the MMA are dims d / d + 1
#pragma unroll
                for (int e = 0; e < kE; ++e)
                    *reinterpret_cast<float2*>(to + (HG == 4 ? j : 2 * j + e) * D + d) = make_float2(o[b][m][e] * even, o[b][m][kO / 2 + e] * odd);
            }
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 4);
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 8);
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 16);
            if (!whole && n == 0) {
                s_frag.m[slot][HG == 4 ? j : 2 * j + e] = m_ref[e];
                s_frag.l[slot][HG == 4 ? j : 2 * j + e] = l_run[e];
            }
        }
        if (!whole && lane == 0) {
            s_frag.seg[slot] = s;
            s_frag.used[slot] = 1;
        }
        __syncwarp();
        if (whole) {
            const int quads = s.heads * (D / 4);
#pragma unroll
            for (int x0 = 0; x0 < HG * (D / 4); x0 += 32) {
                const int x = x0 + lane, h = x / (D / 4);
                const float l0 = __shfl_sync(0xffffffffu, l_run[0], h / kE), l1 = __shfl_sync(0xffffffffu, l_run[kE - 1], h / kE);
                if (x0 < quads) write_quad<NB>(a, s, x, x < quads, reinterpret_cast<const float4*>(to)[x], (h % kE) ? l1 : l0);
            }
            __syncwarp();
        }
    }
    finish<NB>(a, s_frag, [&](int c, int x) { return reinterpret_cast<const float4*>(fragment(c))[x]; });
    write_empty<NB>(a);
}

template <int NB, int HG>
int launch(const PagedArgs& a, cudaStream_t s) {
    if (int st = allow_shared<paged_mma_kernel<NB, HG>>(Plan<NB, HG>::kBytes)) return st;
    paged_mma_kernel<NB, HG><<<148 * Plan<NB, HG>::kCtas, kWorkThreads, Plan<NB, HG>::kBytes, s>>>(a);
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
