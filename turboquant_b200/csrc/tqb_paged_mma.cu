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
//   2^(kShift + kLazy), as high as f16 allows, so that it holds products with small weights and small scales: rms errors of
//   700 tokens stay below 3e-4 down to scales of 3e-7 (with kShift 6: 1.2e-3 at 1e-6, 4.4e-3 at 3e-7).
// O^T = V^T P' (mma.sync f16, K = 16 tokens): P' = p |s_v|, rounded to f16 (once for p, once for the product: 2^-11 each,
//   below the rounding of a bf16 output and within that of f16).  Up to four heads, the two columns of a head carry the
//   scales of two neighbouring blocks, one half2 product for both, and one movmatrix turns them into B fragments.
//   The codes of V enter as SUBNORMAL f16 values c 2^-23 and c 2^-19 - one mask a register, no arithmetic - and the centre 7.5
//   is taken off by starting each accumulation at -7.5 sum P', itself an MMA with constant rows.  Accumulators live for
//   32 tokens and are then added to the running output in rounded f32 additions; one long chain would add up the truncation
//   of the MMA's adder relative to 7.5 sum P'.
//   Where some |s_v| is above 1, so that a product could leave f16, the warp lowers kShift by as much (most often with the
//   first step's maximum, where that costs nothing).
//
// Measured (8 KV heads, head_dim 128, 4 bits, bf16): 64 requests of 8,192 tokens, four query heads a KV head 101.5 us (6.0 TB/s, 0.91
// of a copy); 64 of 531 to 8,192 tokens 43.9 us (of which 6 us until the first products and 5 for the joins); one of 131,072
// tokens 36.9 us.  What binds then is HBM.  Eight query heads 59 us and 50 us: instructions, on 12 warps an SM (registers and
// shared memory); three bits 72 us, 97 requests of up to 2,003 tokens 39.4 us: instructions, twice as many a token as with four
// bits, for codes that cross words and whose centroids come out of tables.
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
constexpr float kShift = 11.0f, kLazy = 4.0f;
constexpr uint32_t kScaleTop = 0x3c003c00u;   // 2^(15 - kShift - kLazy) = 1, twice
constexpr uint32_t kSignBits = 0xB1A6D4B2u;   // bit d: dim d of a block changes its sign (src/cache/precomputed/rotation.rs:16-20)
constexpr float kQMax = 32639.0f;   // 127 * 256 + 127

// A token's NB scales, two a word.
template <int NB, int OFF>
__device__ __forceinline__ void load_scales(uint32_t at, uint32_t (&w)[NB / 2]) {
    if constexpr (NB == 2) {
        w[0] = lds32_o<OFF>(at);
    } else {
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) {
            const uint2 v = i == 0 ? lds64_o<OFF>(at) : lds64_o<OFF + 8>(at);
            w[2 * i] = v.x;
            w[2 * i + 1] = v.y;
        }
    }
}

// x[i]: half2 of code i of the two tokens in the halves of w, as the subnormals c 2^-23 (i even), c 2^-19 (i odd).
__device__ __forceinline__ void codes_to_subnormals(uint32_t w, uint32_t (&x)[4]) {
    const uint32_t w1 = w << 1, w7 = w >> 7;
    x[0] = w1 & 0x001e001eu;
    x[1] = w1 & 0x01e001e0u;
    x[2] = w7 & 0x001e001eu;
    x[3] = w7 & 0x01e001e0u;
}
// Eight 3-bit codes (24 bits; what is above them does not matter) -> a nibble each, the top bit clear.
__device__ __forceinline__ uint32_t nibbles_of_codes(uint32_t w) {
    const uint32_t a = bit_select(w, w << 4, 0x00000fffu);
    const uint32_t b = bit_select(a, a << 2, 0x003f003fu);
    return bit_select(b, b << 1, 0x07070707u) & 0x77777777u;
}
// The bytes of (lo, hi) that the low four nibbles of c, 0 .. 7 each, name.
__device__ __forceinline__ uint32_t byte_of_table(uint32_t lo, uint32_t hi, uint32_t c) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;\n" : "=r"(d) : "r"(lo), "r"(hi), "r"(c));
    return d;
}
constexpr uint32_t kCentreEven = 0x800f800fu;   // -7.5 2^-23 as a subnormal f16, twice
constexpr uint32_t kCentreOdd = 0x80f080f0u;    // -7.5 2^-19

__device__ __forceinline__ uint32_t product(uint32_t a, uint32_t b) { return h2_as_u32(__hmul2(u32_as_h2(a), u32_as_h2(b))); }

template <int NB, int HG, int BITS>
struct Shape {
    static constexpr int kRow = 4 * BITS * NB;          // bytes of a token's codes
    static constexpr int kIdx = kGroupTokens * kRow;    // of a stage's K (or V) codes
    static constexpr int kSc = 2 * NB;                  // of a token's scales
    static constexpr int kOut = HG * NB * 32 * 4;       // of a segment's outputs: they must fit into half a ring
    static constexpr int kUsed = 2 * kIdx + 2 * kGroupTokens * kSc;   // [K codes][V codes][K scales][V scales]
    static constexpr int kStage = kUsed > kOut / kInFlight ? kUsed : kOut / kInFlight;
    static constexpr int kWarpRing = kRing * kStage;      // of a warp
    static constexpr int kCopies = (kIdx / 16 + 31) / 32;   // 16-byte pieces of K (or V) codes that a lane copies, at most
    // 4-bit: 16-byte piece c of token row t lies at piece c ^ swizzle(t), so that the eight rows of an ldmatrix hit different
    // banks.  3-bit rows lie densely: their 6, 12 or 24 words spread over the banks by themselves.
    __device__ static __forceinline__ int swizzle(int t) { return NB == 2 ? (t >> 2) & 1 : NB == 4 ? (t >> 1) & 3 : t & 7; }
};

template <int NB, int HG, int BITS>
struct Plan {
    using G = Shape<NB, HG, BITS>;
    static constexpr int kSets = HG == 4 && BITS == 4 ? 1 : 2;    // sets of digits (3-bit: see the scores)
    static constexpr int kFragment = G::kOut;
    static constexpr int kDigits = kSets * NB * 32 * 8;           // the queries' MMA fragments
    static constexpr int kQueries = HG * NB * 32 * 2;             // the next segment's queries as they are
    static constexpr int kWarpBytes = G::kWarpRing + kFragment + kDigits + kQueries;   // [ring][fragment that began before][digits][queries]
    static constexpr int kBytes = kWorkWarps * kWarpBytes;
    // CTAs of an SM: by shared memory, and three, so that registers hardly spill and fewer parts are joined (head_dim 256: two, and
    // with more than four heads only one has room).
    // 64 requests of 531 to 8,192 tokens, four heads: 43.9 us; with two 46.7, with four 45.2; head_dim 64 32.8, with five 33.8.
    static constexpr int kByShared = 228 * 1024 / (kBytes + 1024 + 2560 + (BITS == 3 ? 8192 : 0)), kByRegs = NB == 8 ? 2 : 3;
    static constexpr int kCtas = kByShared < kByRegs ? kByShared : kByRegs;
};

template <int NB, int HG, int BITS>
__global__ void __launch_bounds__(kWorkThreads, Plan<NB, HG, BITS>::kCtas) paged_mma_kernel(const __grid_constant__ PagedArgs a) {
    using G = Shape<NB, HG, BITS>;
    using L = Plan<NB, HG, BITS>;
    constexpr int D = NB * 32, kE = HG == 4 ? 1 : 2, kPairs = NB / 2;
    constexpr int kO = HG == 4 ? 2 : 4;               // outputs that a lane holds of an MMA tile
    extern __shared__ __align__(128) unsigned char s_dyn[];
    __shared__ Fragments s_frag;
    __shared__ Segment s_next[kWorkWarps];

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = lane >> 2, j = lane & 3;
    __shared__ uint32_t s_pairs[BITS == 3 ? 64 : 1][32];   // half2(value of code i & 7, value of code i >> 3), a copy for each bank
    const float step = 2.0f * a.cent[15] / 15.0f;          // 4-bit: between centroids
    unsigned char* const s_warp = s_dyn + warp * L::kWarpBytes;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_warp);
    unsigned char* const s_digits = s_warp + G::kWarpRing + L::kFragment;
    const uint32_t digits = (uint32_t)__cvta_generic_to_shared(s_digits) + lane * 8;
    const uint32_t halves = 2 * ring + kInFlight * G::kStage;   // (one half's address) + (the other's)
    unsigned char* const s_queries = s_digits + L::kDigits;
    const uint32_t queries = (uint32_t)__cvta_generic_to_shared(s_queries);
    static_assert(kRing == 2 * kInFlight && kStepGroups == kInFlight, "the ring has two halves of a step each");
    static_assert(L::kFragment <= kInFlight * G::kStage && G::kStage % 16 == 0, "what lies in the ring when it is idle does not fit");
    // a fragment's outputs [HG][D]: that of the warp's last segment lies in its idle ring
    auto fragment = [&](int slot) { return reinterpret_cast<float*>(s_dyn + (slot >> 1) * L::kWarpBytes + ((slot & 1) ? 0 : G::kWarpRing)); };
    // ldmatrix: lane l gives the row address of token 8 ((l >> 3) & 1) + (l & 7), block 2 pair + (l >> 4)
    const int tok = 8 * ((lane >> 3) & 1) + (lane & 7);
    const uint32_t off_k = tok * G::kRow + (((lane >> 4) ^ G::swizzle(tok)) << 4);   // ^ 32 pair
    const uint32_t off_s = 2 * G::kIdx + n * G::kSc;
    const int piece_t = lane / NB, piece_c = lane % NB;
    const uint32_t off_p = BITS == 4 ? piece_t * G::kRow + ((piece_c ^ G::swizzle(piece_t)) << 4) : lane * 16;
    // 3-bit: K codes 8j .. 8j + 7 are the 24 bits at byte 3j of a block, V codes 4n .. 4n + 3 the 12 bits at bit 12 n
    const uint32_t off_k3 = n * G::kRow + 4 * ((3 * j) >> 2), off_k3h = off_k3 + (j < 3 ? 4 : 0), sh_k3 = ((3 * j) & 3) * 8;
    const uint32_t off_v3 = G::kIdx + 2 * j * G::kRow + 4 * ((12 * n) >> 5), sh_v3 = (12 * n) & 31, off_v3h = off_v3 + (sh_v3 > 20 ? 4 : 0);
    // those of the other token, three bits up: from bit 12 n - 3 on (n = 0: the word before; what comes from there is masked)
    const int bit_w3 = 12 * n - 3;
    const uint32_t off_w3 = G::kIdx + (2 * j + 1) * G::kRow + 4 * (bit_w3 >> 5), sh_w3 = bit_w3 & 31, off_w3h = off_w3 + (sh_w3 > 17 ? 4 : 0);
    const uint32_t off_ps = 2 * G::kIdx + lane * G::kSc;   // K scales of tokens 0..15, V scales behind them
    const int mask = (1 << a.page_shift) - 1;
    auto pair_of = [&](uint32_t at) {   // table entry, in bits 7 .. 12 of `at`
        return *reinterpret_cast<const uint32_t*>(reinterpret_cast<const unsigned char*>(s_pairs) + bit_select(at, lane * 4, 0x1f80u));
    };

    if (BITS == 3)
        for (int i = threadIdx.x; i < 64 * 32; i += kWorkThreads)
            s_pairs[i >> 5][i & 31] = h2_as_u32(__floats2half2_rn(a.values[(i >> 5) & 7], a.values[i >> 8]));
    if (threadIdx.x < 2 * kWorkWarps) s_frag.used[threadIdx.x] = 0;
    WorkLine line(a);   // (its barriers stand before the first use of what is set above)

    // ---- copies: segment after segment without a break, a step ahead of the products ----
    Segment s{};
    int to_copy = 0, copy_end = 0;            // of the segment whose copies are being made
    int page_now = 0, page_next = 0, page0 = 0;   // pages page0 + 32 k + lane of it, for this k and the next
    const int32_t* table = a.table;
    uint32_t head = 0;
    bool fresh = true;                        // its first group is still to come
    bool bad_copy = false;                    // some page of it does not exist (of those looked at so far)
    const uint8_t *kp = a.kb, *vp = a.vb;
    const uint16_t* sp = a.ks;
    auto page_at = [&](int i) {
        const int page = table[min(page0 + i, (copy_end - 1) >> a.page_shift)];
        const bool bad = (unsigned)page >= (unsigned)a.num_pages;
        bad_copy |= __any_sync(0xffffffffu, bad) != 0;
        return bad ? 0 : page;
    };
    auto open = [&](const Segment& x) {
        to_copy = x.t0;
        copy_end = x.t1;
        page0 = x.t0 >> a.page_shift;
        table = a.table + (size_t)x.req * a.table_stride;
        head = (uint32_t)x.kvh << a.page_shift;
        bad_copy = false;
        fresh = true;
        // the queries ride along with the first group
        const uint8_t* q = reinterpret_cast<const uint8_t*>(a.q) + ((size_t)known_row(a, x.req) * a.q_stride + (size_t)x.head0 * D) * 2;
#pragma unroll
        for (int i = 0; i < (L::kQueries / 16 + 31) / 32; ++i) {
            const int piece = 32 * i + lane;
            if (piece < x.heads * NB * 4) cp_async16(queries + piece * 16, q + piece * 16);
        }
        page_now = page_at(lane);
        page_next = (copy_end - 1) >> a.page_shift >= page0 + 32 ? page_at(32 + lane) : 0;
    };
    auto fill = [&](uint32_t st) {
        if (to_copy < copy_end) {
            const int i = (to_copy >> a.page_shift) - page0;
            if ((to_copy & mask) == 0 || fresh) {
                fresh = false;
                if (i > 0 && (i & 31) == 0) {
                    page_now = page_next;
                    page_next = page_at(i + 32 + lane);
                }
                const int page = __shfl_sync(0xffffffffu, page_now, i & 31);
                const uint32_t row = (((uint32_t)page * a.hkv) << a.page_shift) + head + (to_copy & mask);
                kp = a.kb + (size_t)row * G::kRow + lane * 16;
                vp = a.vb + (size_t)row * G::kRow + lane * 16;
                sp = (lane < 16 ? a.ks : a.vs) + (size_t)(row + (lane & 15)) * NB;
            }
            // whole groups, also where the request ends inside: the page has the room
#pragma unroll
            for (int p = 0; p < G::kCopies; ++p) {
                const uint32_t d = st + (BITS == 4 && NB == 8 && (p & 1) ? off_p ^ 64 : off_p) + p * 512;
                if (G::kIdx / 16 >= 32 * (p + 1) || lane + 32 * p < G::kIdx / 16) {
                    cp_async16(d, kp + p * 512);
                    cp_async16(d + G::kIdx, vp + p * 512);
                }
            }
            cp_async_ca<G::kSc>(st + off_ps, sp);
            kp += G::kIdx;
            vp += G::kIdx;
            sp += kGroupTokens * NB;
        }
        cp_async_commit();
        to_copy += kGroupTokens;
    };

    // One more turn than there are segments: the first has nothing to work on and begins the copies.  (What is written once
    // here is fetched once: a second copy of this code costs a short call more than the turn.)
    uint32_t st = ring;
    for (bool have = false;; have = true) {
        // ---- the next segment; copies go over to it by themselves ----
        bool bad = bad_copy;                  // of this segment
        Segment next{};
        const bool more = line.next(next);
        if (!have && !more) break;
        __syncwarp();                         // (s_next has been read)
        if (lane == 0) s_next[warp] = next;
        bool ahead = false;                   // copies have gone over
        if (have) cp_async_wait<kInFlight - 1>();   // the first group, and the queries
        __syncwarp();
        // ---- queries: rotated, scaled to integers, cut into digits ----
        float qsc[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) qsc[e] = 0.0f;
        if (have) {
            // A lane takes 16 dims of a block: four stages of the butterfly are its own, one is a shuffle away, and its digits are 16
            // bytes of each of the fragments.  (A dim a lane, 80 shuffles and 32 byte stores a segment: 2.7 us instead of 1.2.)
            const float inv_sqrt = 1.0f / sqrtf((float)kBlock);
            constexpr int kHeads = 16 / NB;       // of a pass
            const int b = (lane >> 1) % NB, part = lane & 1;
            const uint32_t neg = kSignBits >> (16 * part);
#pragma unroll 1
            for (int h0 = 0; h0 < HG; h0 += kHeads) {
                const int h = h0 + (lane >> 1) / NB;
                uint4 raw[2];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    raw[k] = h < s.heads ? *reinterpret_cast<const uint4*>(s_queries + (h * D + b * 32 + part * 16 + 8 * k) * 2) : make_uint4(0u, 0u, 0u, 0u);
                float v[16];
                const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = __half22float2(u32_as_h2(w[i]));
                    const bool half = a.q_dtype == TQB_F16;
                    v[2 * i] = half ? f.x : __uint_as_float(w[i] << 16);
                    v[2 * i + 1] = half ? f.y : __uint_as_float(w[i] & 0xffff0000u);
                }
#pragma unroll
                for (int m = 1; m < 16; m <<= 1)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if ((i & m) == 0) {
                            const float x = v[i], y = v[i + m];
                            v[i] = x + y;
                            v[i + m] = x - y;
                        }
                uint32_t top = 0;   // of the bits, so that NaN is above infinity
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float other = __shfl_xor_sync(0xffffffffu, v[i], 1);
                    v[i] = (part ? other - v[i] : v[i] + other) * inv_sqrt * a.sign_mag;
                    top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
                    v[i] = __uint_as_float(__float_as_uint(v[i]) ^ ((neg << (31 - i)) & 0x80000000u));
                }
#pragma unroll
                for (int o = 1; o < 2 * NB; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                float m = __uint_as_float(top);
                if (!(m <= FLT_MAX)) m = __uint_as_float(0x7fc00000u);   // not finite: every score is NaN
                float inv = m > 0.0f ? kQMax / m : 0.0f;
                if (!(inv <= FLT_MAX)) inv = 0.0f;                       // the largest component is below 1e-34, or not finite
                // x = 256 hi + lo, both signed: hi is byte 1 of x + 128.  Fragment (b, 4n' + j') of column n' has eight dims from
                // 32 b + 8 j' on, a byte each.  4-bit: the even ones (k-slots 4j' ..) in its first word, the odd ones (k-slots
                // 16 + 4j' ..) in the second; 3-bit: the first four, the last four.
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = (uint32_t)__float2int_rn(v[BITS == 4 ? 8 * (k >> 1) + 2 * i + (k & 1) : 4 * k + i] * inv);
                    lo[k] = __byte_perm(__byte_perm(x[0], x[1], 0x0040), __byte_perm(x[2], x[3], 0x0040), 0x5410);
                    hi[k] = __byte_perm(__byte_perm(x[0] + 128u, x[1] + 128u, 0x0051), __byte_perm(x[2] + 128u, x[3] + 128u, 0x0051), 0x5410);
                }
                const uint4 hi4 = make_uint4(hi[0], hi[1], hi[2], hi[3]), lo4 = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if (h < HG) {
                    unsigned char* const at = s_digits + b * 256 + part * 16;   // column 0
                    if (HG == 4) {
                        *reinterpret_cast<uint4*>(at + 2 * h * 32) = hi4;
                        *reinterpret_cast<uint4*>(at + (2 * h + 1) * 32) = lo4;
                        if (BITS == 3) {
                            *reinterpret_cast<uint4*>(at + NB * 256 + 2 * h * 32) = make_uint4(0u, 0u, 0u, 0u);
                            *reinterpret_cast<uint4*>(at + NB * 256 + (2 * h + 1) * 32) = hi4;
                        }
                    } else {
                        *reinterpret_cast<uint4*>(at + h * 32) = hi4;
                        *reinterpret_cast<uint4*>(at + NB * 256 + h * 32) = lo4;
                    }
                }
#pragma unroll
                for (int e = 0; e < kE; ++e) {
                    const int mine = (HG == 4 ? j : 2 * j + e) - h0;   // the lane's head, counted from the pass's first
                    const float mh = __shfl_sync(0xffffffffu, m, mine * 2 * NB);
                    if (mine >= 0 && mine < kHeads)
                        qsc[e] = mh * (a.qk_const * (BITS == 4 ? step / (kQMax * 16.0f) : a.cent[7] * 256.0f / (kQMax * kQMax)));
                }
            }
            __syncwarp();
        }

        float shift = kShift;
        uint32_t sv_limit = kScaleTop;
        float m_ref[kE], l_run[kE];
        float o[NB][2][kO];
        {
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
            for (int t0 = s.t0; !have || t0 < s.t1; t0 += kStepGroups * kGroupTokens) {
                const uint32_t st_other = halves - st;
                if (to_copy >= copy_end && more && !ahead) {   // this segment's copies are under way: the next one's
                    bad |= bad_copy;
                    ahead = true;
                    open(s_next[warp]);
                }
#pragma unroll
                for (int u = 0; u < kStepGroups; ++u) fill(st_other + u * G::kStage);
                if (!have) {
                    st = st_other;
                    break;
                }
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
                    uint32_t ks[2][kPairs];   // scales of tokens n, n + 8
                    load_scales<NB, 0>(stu + off_s, ks[0]);
                    load_scales<NB, 8 * G::kSc>(stu + off_s, ks[1]);
                    static_for<0, kPairs>([&](auto p_) {
                        constexpr int p = decltype(p_)::value;
                        uint32_t kw[4];
                        if (BITS == 4) ldsm4_o<0>(stu + (off_k ^ (32 * p)), kw);
                        const uint32_t sa = ks[0][p] & 0x7fff7fffu, sb = ks[1][p] & 0x7fff7fffu;
                        static_for<0, 2>([&](auto i_) {
                            constexpr int i = decltype(i_)::value, b = 2 * p + i;
                            const float ka = i ? __high2float(u32_as_h2(sa)) : __low2float(u32_as_h2(sa));
                            const float kc = i ? __high2float(u32_as_h2(sb)) : __low2float(u32_as_h2(sb));
                            const uint2 qa = lds64_o<b * 256>(digits);
                            int hi[4], lo[4];
                            if constexpr (BITS == 4) {
                                // c ^ 8 is the two's complement of c - 8; at the top of a byte with bit 3 set below it: 16 (c - 7.5)
                                const uint32_t u0 = kw[2 * i], u1 = kw[2 * i + 1];
                                const uint32_t a0 = lop3_xor_select(u0 << 4, 0xF0F0F0F0u, 0x88888888u), a2 = lop3_xor_select(u0, 0xF0F0F0F0u, 0x88888888u);
                                const uint32_t a1 = lop3_xor_select(u1 << 4, 0xF0F0F0F0u, 0x88888888u), a3 = lop3_xor_select(u1, 0xF0F0F0F0u, 0x88888888u);
                                imma16832(hi, a0, a1, a2, a3, qa.x, qa.y);
                                if (HG == 8) {
                                    const uint2 qb = lds64_o<(HG == 8 ? NB + b : b) * 256>(digits);
                                    imma16832(lo, a0, a1, a2, a3, qb.x, qb.y);
                                }
                            } else {
                                // The centroid as two base-256 digits: its bytes come out of an eight-entry table by PRMT.  Two columns a
                                // head: the second set of digits has D1 in D0's column, so that one accumulator gathers what counts 256.
                                uint32_t x[2][4];   // [token n | n + 8]: first digits of codes 0..3, 4..7, second digits
                                static_for<0, 2>([&](auto t_) {
                                    constexpr int t = decltype(t_)::value;
                                    const uint32_t c = nibbles_of_codes(__funnelshift_r(lds32_o<12 * b + 8 * t * G::kRow>(stu + off_k3), lds32_o<12 * b + 8 * t * G::kRow>(stu + off_k3h), sh_k3));
                                    x[t][0] = byte_of_table(a.digits[0], a.digits[1], c);
                                    x[t][1] = byte_of_table(a.digits[0], a.digits[1], c >> 16);
                                    x[t][2] = byte_of_table(a.digits[2], a.digits[3], c);
                                    x[t][3] = byte_of_table(a.digits[2], a.digits[3], c >> 16);
                                });
                                const uint2 qb = lds64_o<(NB + b) * 256>(digits);
                                imma16832(hi, x[0][0], x[1][0], x[0][1], x[1][1], qa.x, qa.y);
                                if (HG == 4) {
                                    imma16832_acc(hi, x[0][2], x[1][2], x[0][3], x[1][3], qb.x, qb.y);
                                } else {
                                    imma16832(lo, x[0][0], x[1][0], x[0][1], x[1][1], qb.x, qb.y);
                                    imma16832_acc(lo, x[0][2], x[1][2], x[0][3], x[1][3], qa.x, qa.y);
                                }
                            }
                            if constexpr (HG == 4) {
                                acc[0][0] = fmaf(ka, (float)(hi[0] * 256 + hi[1]), acc[0][0]);
                                acc[1][0] = fmaf(kc, (float)(hi[2] * 256 + hi[3]), acc[1][0]);
                            } else {
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
                if (!ahead) bad |= bad_copy;
                if (bad || t0 + kStepGroups * kGroupTokens > s.t1) {
#pragma unroll
                    for (int u = 0; u < kStepGroups; ++u) {
                        const int gs = t0 + u * kGroupTokens;
                        const bool none = bad && (unsigned)a.table[s.req * a.table_stride + (min(gs, s.t1 - 1) >> a.page_shift)] >= (unsigned)a.num_pages;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            if (none || gs + n + 8 * t >= s.t1) {
                                out[u][t] = true;
                                sv_mask[u][t] = 0u;
                            }
                    }
                }
                // ---- scales of V, and the largest of them ----
                uint32_t sv[kStepGroups][2][kPairs], sv_top = 0u;
                static_for<0, kStepGroups>([&](auto u_) {
                    constexpr int u = decltype(u_)::value;
                    static_for<0, 2>([&](auto t_) {
                        constexpr int t = decltype(t_)::value;
                        load_scales<NB, 16 * G::kSc + 8 * t * G::kSc>(st + u * G::kStage + off_s, sv[u][t]);
                        static_for<0, kPairs>([&](auto p_) {
                            constexpr int pr = decltype(p_)::value;
                            sv[u][t][pr] &= sv_mask[u][t];
                            sv_top = h2_as_u32(__hmax2(u32_as_h2(sv_top), u32_as_h2(sv[u][t][pr])));
                        });
                    });
                });
                // ---- softmax ----
                float x[kStepGroups][2][kE];
                bool over = ((sv_limit - sv_top) & 0x80008000u) != 0u;   // some half of sv_top is larger (a borrow is one itself)
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
                    const uint32_t largest = __reduce_max_sync(0xffffffffu, max(sv_top & 0xffffu, sv_top >> 16));
                    float less = 0.0f;
                    if (largest > (sv_limit & 0xffffu)) {   // (f16 bits, positive: they compare like numbers)
                        const uint32_t above = min((largest - (sv_limit & 0xffffu) + 1023u) >> 10, (0x7c00u - (sv_limit & 0xffffu)) >> 10);
                        less = (float)above;                // powers of two
                        shift -= less;
                        sv_limit += above * 0x04000400u;
                    }
#pragma unroll
                    for (int e = 0; e < kE; ++e) {   // (products rounded as in their maximum, which rounded up keeps x at shift or below: scores may be 2^27 and more)
                        float mx = -INFINITY;
#pragma unroll
                        for (int u = 0; u < kStepGroups; ++u)
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                if (!out[u][t]) mx = fmaxf(mx, raw[u][t][e] * qsc[e]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float m_new = fmaxf(m_ref[e] + less, __fadd_ru(mx, -shift)), keep = ex2(m_ref[e] - m_new);
                        m_ref[e] = m_new;
                        l_run[e] *= keep;
#pragma unroll
                        for (int u = 0; u < kStepGroups; ++u)
#pragma unroll
                            for (int t = 0; t < 2; ++t) x[u][t][e] = out[u][t] ? -INFINITY : raw[u][t][e] * qsc[e] - m_new;
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
                            const uint32_t w = sv[u][t][pr];
                            if constexpr (HG == 4) {   // columns 2j, 2j + 1: head j with the scales of blocks 2 pr, 2 pr + 1
                                pq[u][pr][t] = movmatrix_trans(product(ph, w));
                            } else {                   // columns 2j, 2j + 1: heads 2j, 2j + 1
                                pq[u][2 * pr][t] = movmatrix_trans(product(ph, h2_as_u32(__low2half2(u32_as_h2(w)))));
                                pq[u][2 * pr + 1][t] = movmatrix_trans(product(ph, h2_as_u32(__high2half2(u32_as_h2(w)))));
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
                    for (int u = 0; u < kStepGroups; ++u)
                        if (BITS == 4) ldsm4t_o<G::kIdx>(st + u * G::kStage + (off_k ^ (32 * pr)), vw[u]);
                    float centre[4];
                    static_for<0, 2>([&](auto i_) {
                        constexpr int i = decltype(i_)::value, b = 2 * pr + i, f = HG == 4 ? pr : b;
                        if (BITS == 3) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) centre[k] = 0.0f;
                        } else if (HG == 8 || i == 0) {
                            mma16816_from(centre, zero, kCentreEven, kCentreOdd, kCentreEven, kCentreOdd, pq[0][f][0], pq[0][f][1]);
#pragma unroll
                            for (int u = 1; u < kStepGroups; ++u)
                                mma16816(centre, kCentreEven, kCentreOdd, kCentreEven, kCentreOdd, pq[u][f][0], pq[u][f][1]);
                        }
                        float acc[2][4];
                        static_for<0, kStepGroups>([&](auto u_) {
                            constexpr int u = decltype(u_)::value;
                            uint32_t xa[4], xb[4];   // tokens 2j, 2j + 1 and 2j + 8, 2j + 9: codes 4n .. 4n + 3 of the block
                            if constexpr (BITS == 4) {
                                codes_to_subnormals(vw[u][2 * i], xa);
                                codes_to_subnormals(vw[u][2 * i + 1], xb);
                            } else {
                                static_for<0, 2>([&](auto o_) {
                                    constexpr int o8 = decltype(o_)::value, off = 12 * b + 8 * o8 * G::kRow + u * G::kStage;
                                    const uint32_t ya = __funnelshift_r(lds32_o<off>(st + off_v3), lds32_o<off>(st + off_v3h), sh_v3);
                                    const uint32_t yb = __funnelshift_r(lds32_o<off>(st + off_w3), lds32_o<off>(st + off_w3h), sh_w3);
                                    // six-bit pairs (token 2j | token 2j + 1 << 3): codes 0 and 2, codes 1 and 3 (3 bits up)
                                    const uint32_t z0 = bit_select(ya, yb, 0x1c7u), z1 = bit_select(ya, yb, 0xe38u);
                                    uint32_t* x = o8 == 0 ? xa : xb;
                                    x[0] = pair_of(z0 << 7);
                                    x[1] = pair_of(z1 << 4);
                                    x[2] = pair_of(z0 << 1);
                                    x[3] = pair_of(z1 >> 2);
                                });
                            }
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                if (u == 0) mma16816_from(acc[m], centre, xa[2 * m], xa[2 * m + 1], xb[2 * m], xb[2 * m + 1], pq[u][f][0], pq[u][f][1]);
                                else mma16816(acc[m], xa[2 * m], xa[2 * m + 1], xb[2 * m], xb[2 * m + 1], pq[u][f][0], pq[u][f][1]);
                            }
                        });
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int k = 0; k < kO; ++k) o[b][m][k] += HG == 4 ? acc[m][2 * k + i] : acc[m][k];
                    });
                });
                __syncwarp();   // the stages may be filled again
                st = st_other;
            }
        }

        if (!have) {
            s = s_next[warp];
            continue;
        }
        // ---- the segment's end ----
        // A whole segment's outputs pass through the half of the ring that holds nothing yet: the copies in flight are in `st`.
        const bool whole = s.whole();
        const int slot = 2 * warp + (s.begins ? 1 : 0);
        float* const to = whole ? reinterpret_cast<float*>(s_warp + (halves - st - ring)) : fragment(slot);
        if (!whole && s.begins) cp_async_wait<0>();   // the warp's last segment: its ring is idle
        const float even = BITS == 4 ? step * 8388608.0f : a.kappa, odd = BITS == 4 ? step * 524288.0f : a.kappa;   // 2^23, 2^19
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
#pragma unroll 1
            for (int x0 = 0; x0 < quads; x0 += 32) {
                const int x = x0 + lane, h = x / (D / 4);
                const float l0 = __shfl_sync(0xffffffffu, l_run[0], h / kE), l1 = __shfl_sync(0xffffffffu, l_run[kE - 1], h / kE);
                write_quad(a.out, a.out_dtype, quad_at<NB>(a, s, x), x < quads, reinterpret_cast<const float4*>(to)[x], (h % kE) ? l1 : l0, a.sign_mag);
            }
            __syncwarp();
        }
        if (!more) break;
        s = s_next[warp];
    }
    finish<NB>(a, s_frag, [&](int c, int x) { return reinterpret_cast<const float4*>(fragment(c))[x]; });
    write_empty<NB>(a);
}

template <int NB, int HG, int BITS>
int launch(const PagedArgs& a, cudaStream_t s) {
    using L = Plan<NB, HG, BITS>;
    if (int st = allow_shared<paged_mma_kernel<NB, HG, BITS>>(L::kBytes)) return st;
    paged_mma_kernel<NB, HG, BITS><<<148 * L::kCtas, kWorkThreads, L::kBytes, s>>>(a);
    return check_launch(s);
}

template <int BITS>
int launch_bits(const PagedArgs& a, int head_dim, cudaStream_t s) {
    const bool narrow = a.group <= 4;
    if (head_dim == 64) return narrow ? launch<2, 4, BITS>(a, s) : launch<2, 8, BITS>(a, s);
    if (head_dim == 128) return narrow ? launch<4, 4, BITS>(a, s) : launch<4, 8, BITS>(a, s);
    return narrow ? launch<8, 4, BITS>(a, s) : launch<8, 8, BITS>(a, s);
}

}  // namespace

int launch_paged_mma(const PagedArgs& a, int head_dim, int bits, cudaStream_t s) {
    if (bits == 4) return launch_bits<4>(a, head_dim, s);
    PagedArgs b = a;
    if (!pqo3_values(TQB_MAXNORM, true, b.kappa, b.values)) return TQB_ERR_UNSUPPORTED;
    for (int i = 0; i < 4; ++i) b.digits[i] = 0;
    for (int i = 0; i < 8; ++i) {
        const int v = (int)lrintf(a.cent[i] / a.cent[7] * kQMax), lo = (int)(signed char)(v & 0xff), hi = (v - lo) >> 8;
        b.digits[i >> 2] |= (uint32_t)(hi & 0xff) << (8 * (i & 3));
        b.digits[2 + (i >> 2)] |= (uint32_t)(lo & 0xff) << (8 * (i & 3));
    }
    return launch_bits<3>(b, head_dim, s);
}

}  // namespace tqb
