// Paged cache: block tables and slot maps from lengths, the rows that go into pages (norm, rotation and packing in one pass)
// and the rows that come back from them.  The attention over the pages is in tqb_paged_attention.cu.
#include "tqb_common.cuh"
#include "tqb_paged.cuh"
#include "tqb_pqo_quant.cuh"

namespace tqb {
namespace {

// ---- block tables, slots and positions of a step ----------------------------------------------------------------------
// need_r = ceil((s_r + n_r) / P) - ceil(s_r / P); page i of them is free[F - 1 - (start_r + i)], start the exclusive sum of
// need.  Every CTA does the two prefix sums over the requests for itself (8 bytes a request from L2) and then takes its
// share of the tokens and of the new table entries; nobody waits for anybody.  What may be updated in place - lengths and
// state - is written by the CTA that finishes last, when all have read it.  Bound: launch and two dependent loads.
constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 1024;   // tokens a CTA

struct PlanArgs {
    const int32_t* seq;
    const int32_t* fresh;
    int32_t* table;
    long long table_stride;
    const int32_t* free_pages;
    int32_t* state;
    int64_t* slots;
    int32_t* positions;
    int32_t* cu;
    int32_t* kv_lens;
    int32_t* state_out;
    int requests, max_blocks, page_shift, capacity;
};

__device__ __forceinline__ long long pages_of(long long tokens, int shift) { return (tokens + (1ll << shift) - 1) >> shift; }

// largest i in [0, n] with v[i] <= x; v[0] = 0 <= x
__device__ __forceinline__ int last_not_above(const int* v, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Exclusive sums of (a, b) over the block's threads, in order; returns the totals through ta, tb.
template <int THREADS>
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long& ta, long long& tb) {
    __shared__ long long s_a[THREADS / 32], s_b[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) { a += x; b += y; }
    }
    if (lane == 31) { s_a[warp] = a; s_b[warp] = b; }
    __syncthreads();
    ta = tb = 0;
    long long pa = 0, pb = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w == warp) { pa = ta; pb = tb; }
        ta += s_a[w];
        tb += s_b[w];
    }
    a += pa - a0;
    b += pb - b0;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanArgs a) {
    __shared__ int s_cu[TQB_PAGED_MAX_REQUESTS + 1], s_start[TQB_PAGED_MAX_REQUESTS + 1];
    __shared__ int s_last;
    const int tid = threadIdx.x, R = a.requests, sh = a.page_shift;
    const long long limit = min((long long)a.max_blocks << sh, 0x7fffffffll);
    const long long avail = max(a.state[0], 0);
    const int per = (R + kPlanThreads - 1) / kPlanThreads, r0 = min(tid * per, R), r1 = min(r0 + per, R);
    long long nt = 0, np = 0;
    int bad = 0;
    for (int r = r0; r < r1; ++r) {
        const long long s = a.seq[r], n = a.fresh[r];
        if (s < 0 || n < 0 || s + n > limit) {
            bad = 1;
        } else {
            nt += n;
            np += pages_of(s + n, sh) - pages_of(s, sh);
        }
    }
    bad = __syncthreads_or(bad);
    long long tokens, pages;
    block_scan2<kPlanThreads>(nt, np, tokens, pages);
    const int status = bad ? TQB_PLAN_BAD_LENGTH : tokens > a.capacity ? TQB_PLAN_OVER_CAPACITY : pages > avail ? TQB_PLAN_OUT_OF_PAGES : TQB_PLAN_OK;
    if (status != TQB_PLAN_OK) tokens = pages = 0;   // nothing is planned
    for (int r = r0; r < r1; ++r) {
        s_cu[r] = status == TQB_PLAN_OK ? (int)nt : 0;
        s_start[r] = status == TQB_PLAN_OK ? (int)np : 0;
        if (status == TQB_PLAN_OK) {
            const long long s = a.seq[r], n = a.fresh[r];
            nt += n;
            np += pages_of(s + n, sh) - pages_of(s, sh);
        }
    }
    if (tid == 0) {
        s_cu[R] = (int)tokens;
        s_start[R] = (int)pages;
    }
    __syncthreads();
    const int step = gridDim.x * kPlanThreads, at = blockIdx.x * kPlanThreads + tid;
    for (int t = at; t < a.capacity; t += step) {
        long long slot = -1;
        int pos = 0;
        if (t < (int)tokens) {
            const int r = last_not_above(s_cu, R, t);   // of requests without new tokens the last one that starts here
            const int s = a.seq[r], have = (int)pages_of(s, sh);
            pos = s + (t - s_cu[r]);
            const int b = pos >> sh;
            const int page = b < have ? a.table[r * a.table_stride + b] : a.free_pages[avail - 1 - (s_start[r] + b - have)];
            if (page >= 0) slot = ((long long)page << sh) + (pos & ((1 << sh) - 1));
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
    for (int i = at; i < (int)pages; i += step) {
        const int r = last_not_above(s_start, R, i);
        a.table[r * a.table_stride + pages_of(a.seq[r], sh) + (i - s_start[r])] = a.free_pages[avail - 1 - i];
    }
    for (int r = at; r <= R; r += step) a.cu[r] = s_cu[r];
    if (gridDim.x > 1) {
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            s_last = atomicAdd(reinterpret_cast<unsigned*>(a.state) + 1, 1u) == gridDim.x - 1;
        }
        __syncthreads();
        if (!s_last) return;
    } else {
        __syncthreads();
    }
    for (int r = tid; r < R; r += kPlanThreads) a.kv_lens[r] = status == TQB_PLAN_OK ? a.seq[r] + a.fresh[r] : a.seq[r];
    if (tid == 0) {
        a.state[1] = 0;
        a.state_out[0] = (int)(avail - pages);
        a.state_out[1] = 0;
        a.state_out[2] = status;
        a.state_out[3] = 0;
    }
}

// The pages of finished requests back onto the list, by one CTA: a release is rare and short.
constexpr int kReleaseThreads = 1024;

__global__ void __launch_bounds__(kReleaseThreads) release_kernel(const uint8_t* mask, int32_t* seq, int requests, int32_t* table,
                                                                  long long table_stride, int max_blocks, int32_t* free_pages,
                                                                  int free_capacity, int32_t* state, int sh) {
    __shared__ int s_start[TQB_PAGED_MAX_REQUESTS + 1];
    const int tid = threadIdx.x;
    const long long limit = min((long long)max_blocks << sh, 0x7fffffffll), avail = max(state[0], 0);
    const int per = (requests + kReleaseThreads - 1) / kReleaseThreads, r0 = min(tid * per, requests), r1 = min(r0 + per, requests);
    long long np = 0, unused = 0, pages, unused_total;
    int bad = 0;
    for (int r = r0; r < r1; ++r) {
        if (!mask[r]) continue;
        if (seq[r] < 0 || seq[r] > limit) bad = 1;
        else np += pages_of(seq[r], sh);
    }
    bad = __syncthreads_or(bad);
    block_scan2<kReleaseThreads>(np, unused, pages, unused_total);
    const int status = bad ? TQB_PLAN_BAD_LENGTH : avail + pages > free_capacity ? TQB_PLAN_OUT_OF_PAGES : TQB_PLAN_OK;
    if (status != TQB_PLAN_OK) {
        if (tid == 0) state[2] = status;
        return;
    }
    for (int r = r0; r < r1; ++r) {
        s_start[r] = (int)np;
        if (mask[r]) np += pages_of(seq[r], sh);
    }
    if (tid == 0) s_start[requests] = (int)pages;
    __syncthreads();
    for (int i = tid; i < (int)pages; i += kReleaseThreads) {
        const int r = last_not_above(s_start, requests, i);
        int32_t* e = table + r * table_stride + (i - s_start[r]);
        free_pages[avail + i] = *e;
        *e = -1;
    }
    __syncthreads();
    for (int r = r0; r < r1; ++r)
        if (mask[r]) seq[r] = 0;
    if (tid == 0) {
        state[0] = (int)(avail + pages);
        state[2] = TQB_PLAN_OK;
    }
}

// ---- rows into pages, with norm and rotation ---------------------------------------------------------------------------
// One warp pass takes 32 / (D / 8) heads of a token, eight consecutive elements a lane: every load and store of a warp is
// dense, the norm's sum and the partner of a rotated pair are shuffles away, and the 32-point butterfly runs stages 1, 2, 4
// in the lane and 8, 16 between lanes - the operand pairs of the scalar butterfly, so the codes are those of
// tqb_block_quantize.  The angles of a token are computed once per CTA: position * inv_freq in f64, less whole turns, then
// sincosf in f32 (an f32 product would be off by position * 2^-24, 0.06 rad at a million tokens).
constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;

struct RowSpan {            // one tensor of rows [tokens, heads, head_dim]
    const void* in;
    void* out;
    long long in_token, in_head, out_token, out_head;   // strides in elements
    const void* weight;
    int heads;
};
struct RowArgs {
    RowSpan q, k, v;
    const void* positions;
    const float* inv_freq;
    const int64_t* slots;
    uint8_t* idx[2];        // K, V
    uint16_t* sc[2];
    long long num_slots;
    int tokens, rot_dim, flags, kv_heads, page_shift;
    float eps;
    float outer_centroid;
};

template <typename T>
struct Eight;   // eight elements of a row
template <>
struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        a = make_float4(v[0], v[1], v[2], v[3]);
        b = make_float4(v[4], v[5], v[6], v[7]);
    }
    __device__ __forceinline__ void store(float* p) const {
        *reinterpret_cast<float4*>(p) = a;
        *reinterpret_cast<float4*>(p + 4) = b;
    }
};
template <>
struct Eight<__nv_bfloat16> {
    uint4 r;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        r = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = r; }
};
template <>
struct Eight<__half> {
    uint4 r;
    __device__ __forceinline__ void load(const __half* p) { r = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        r = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void store(__half* p) const { *reinterpret_cast<uint4*>(p) = r; }
};

// The block's 32 values, eight a lane in four neighbouring lanes (quarter: lane & 3) -> this lane's eight codes in the low
// 8 * BITS bits; returns the scale.  Arithmetic and results of pqo_quantize_values.
template <int BITS>
__device__ __forceinline__ float quantize8(float (&v)[8], int quarter, const Codebook& cb, float outer_centroid, uint32_t& codes) {
#pragma unroll
    for (int h = 1; h < 8; h <<= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((i & h) == 0) {
                const float x = v[i], y = v[i + h];
                v[i] = x + y;
                v[i + h] = x - y;
            }
#pragma unroll
    for (int m = 1; m <= 2; m <<= 1) {
        const bool upper = (quarter & m) != 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float other = __shfl_xor_sync(0xffffffffu, v[i], m);
            v[i] = upper ? (other - v[i]) : (v[i] + other);
        }
    }
    const float inv_sqrt = 1.0f / sqrtf((float)kBlock);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2)) * inv_sqrt;
    const float raw = __fdiv_rn(amax, outer_centroid);
    const float scale = raw > kMinNorm ? raw : kMinNorm;
    const float r = __frcp_rn(scale);
    const uint32_t neg = kSignMask >> (8 * quarter);
    codes = 0u;
    if (BITS == 4) {
        const float inv_step = 15.0f / (2.0f * cb.c[15]);
        const float cpos = (inv_sqrt * r) * inv_step;
        const float kMagic = 12582912.0f;   // 1.5 * 2^23
        float far = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float u = fmaf(v[i], ((neg >> i) & 1u) ? -cpos : cpos, 7.5f);
            const float m = u + kMagic;
            far = fmaxf(far, fabsf(u - (m - kMagic)));
            codes |= (__float_as_uint(m) & 15u) << (4 * i);
        }
        if (far > 0.49998f) {   // rare: exact division and the f32 boundary table
            codes = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = __fdiv_rn((v[i] * inv_sqrt) * (((neg >> i) & 1u) ? -1.0f : 1.0f), scale);
                uint32_t c = 0;
#pragma unroll
                for (int k = 0; k < 15; ++k) c += (t > cb.b[k]) ? 1u : 0u;
                codes |= c << (4 * i);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float rot = (v[i] * inv_sqrt) * (((neg >> i) & 1u) ? -1.0f : 1.0f);
            // rot / scale, correctly rounded: the quotient corrected by its remainder (Markstein, IBM J. Res. Dev. 34, 1990)
            const float q = rot * r;
            const float t = fmaf(fmaf(q, -scale, rot), r, q);
            uint32_t c = 0;
#pragma unroll
            for (int k = 0; k < 7; ++k) c += (t > cb.b[k]) ? 1u : 0u;
            codes |= c << (3 * i);
        }
    }
    return scale;
}

template <typename T, int LPH, int BITS>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const __grid_constant__ RowArgs a, const __grid_constant__ Codebook cb) {
    constexpr int D = LPH * 8, HPW = 32 / LPH;
    __shared__ __align__(16) float2 s_cs[2][D / 2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int sub = lane / LPH, l = lane % LPH;
    const int half = a.rot_dim >> 1;
    const bool inter = (a.flags & TQB_ROPE_INTERLEAVED) != 0, norm = (a.flags & TQB_ROPE_NO_NORM) == 0;
    const int heads = a.q.heads + a.k.heads + a.v.heads;
    int par = 0;
    for (int t = blockIdx.x; t < a.tokens; t += gridDim.x, par ^= 1) {
        if (half > 0) {
            if (tid < half) {
                const double pos = (a.flags & TQB_ROPE_POSITIONS_64) ? (double)reinterpret_cast<const long long*>(a.positions)[t]
                                                                    : (double)reinterpret_cast<const int*>(a.positions)[t];
                const double ang = pos * (double)a.inv_freq[tid];
                const double turns = rint(ang * 0.15915494309189535);
                float si, co;
                sincosf((float)fma(turns, -6.283185307179586, ang), &si, &co);
                s_cs[par][tid] = make_float2(co, si);
            }
            __syncthreads();   // one barrier a token: the other half of s_cs is free again when the next but one writes it
        }
        long long slot = -1;
        size_t page = 0;
        int in_page = 0;
        if (BITS != 0) {
            slot = a.slots[t];
            if (slot >= a.num_slots) slot = -1;
            page = (size_t)(slot >> a.page_shift);
            in_page = (int)(slot & ((1 << a.page_shift) - 1));
        }
        for (int g = warp; g * HPW < heads; g += kRowWarps) {
            const bool live = g * HPW + sub < heads;
            const int hd = min(g * HPW + sub, heads - 1);
            const int kind = hd < a.q.heads ? 0 : hd < a.q.heads + a.k.heads ? 1 : 2;
            const RowSpan& s = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
            const int h = kind == 0 ? hd : kind == 1 ? hd - a.q.heads : hd - a.q.heads - a.k.heads;
            float v[8];
            Eight<T> e;
            e.load(reinterpret_cast<const T*>(s.in) + t * s.in_token + h * s.in_head + 8 * l);
            e.get(v);
            // the shuffles below are done by all lanes, whichever tensor their head is of
            if (norm) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (kind != 2) {
                    const float r = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
                    float w[8];
                    if (s.weight != nullptr) {
                        Eight<T> we;
                        we.load(reinterpret_cast<const T*>(s.weight) + 8 * l);
                        we.get(w);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = 1.0f;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = (v[i] * r) * w[i];
                }
            }
            if (half > 0) {
                if (inter) {
                    if (kind != 2 && 8 * l < a.rot_dim) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 cs = s_cs[par][4 * l + i];
                            const float x = v[2 * i], y = v[2 * i + 1];
                            v[2 * i] = fmaf(x, cs.x, -(y * cs.y));
                            v[2 * i + 1] = fmaf(y, cs.x, x * cs.y);
                        }
                    }
                } else {
                    const int hl = half >> 3;   // lanes of half a rotated row
                    const bool first = l < hl, turns = l < 2 * hl;
                    const int from = lane + (!turns ? 0 : first ? hl : -hl);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float other = __shfl_sync(0xffffffffu, v[i], from);
                        if (kind != 2 && turns) {
                            const float2 cs = s_cs[par][8 * (first ? l : l - hl) + i];
                            v[i] = fmaf(v[i], cs.x, first ? -(other * cs.y) : other * cs.y);
                        }
                    }
                }
            }
            e.set(v);
            if (live && s.out != nullptr) e.store(reinterpret_cast<T*>(s.out) + t * s.out_token + h * s.out_head + 8 * l);
            if (BITS != 0) {
                e.get(v);   // keys as their type holds them
                uint32_t codes;
                const float scale = quantize8<BITS == 0 ? 4 : BITS>(v, lane & 3, cb, a.outer_centroid, codes);
                const uint32_t next = BITS == 3 ? __shfl_down_sync(0xffffffffu, codes, 1) : 0u;
                if (live && kind != 0 && slot >= 0) {
                    const size_t row = ((page * a.kv_heads + h) << a.page_shift) + in_page;
                    uint32_t* wp = reinterpret_cast<uint32_t*>(a.idx[kind - 1] + row * (D / 8 * BITS));
                    if (BITS == 4) {
                        wp[l] = codes;
                    } else {
                        const int q = l & 3;   // four lanes' 24 bits make three words
                        if (q < 3) wp[(l >> 2) * 3 + q] = (codes >> (8 * q)) | (next << (24 - 8 * q));
                    }
                    if ((l & 3) == 0) a.sc[kind - 1][row * (D / 32) + (l >> 2)] = f32_to_f16_bits(-scale);   // outlier blocks store -scale
                }
            }
        }
    }
}

// ---- rows back from pages ----------------------------------------------------------------------------------------------
// Eight codes a lane like above; the values and their roundings are those of tqb_block_dequantize.  Bound: HBM (stores).
struct BackArgs {
    const uint8_t* idx[2];
    const uint16_t* sc[2];
    void* out[2];
    const int64_t* slots;
    long long n, num_slots;
    int kv_heads, page_shift;
    float sign_mag;
};

template <typename T, int LPH, int BITS>
__global__ void __launch_bounds__(kRowThreads) back_kernel(const __grid_constant__ BackArgs a, const __grid_constant__ Codebook cb) {
    constexpr int D = LPH * 8, HPW = 32 / LPH, kCodes = 1 << BITS;
    __shared__ float s_tab[kCodes][32];   // a copy of the codebook for each bank
    const int tid = threadIdx.x, lane = tid & 31;
    const int sub = lane / LPH, l = lane % LPH;
    for (int i = tid; i < kCodes * 32; i += kRowThreads) s_tab[i >> 5][i & 31] = cb.c[i >> 5] * a.sign_mag;
    __syncthreads();
    const float inv_sqrt = 1.0f / sqrtf((float)kBlock);
    const uint32_t neg = kSignMask >> (8 * (lane & 3));
    const int side = blockIdx.y;
    const unsigned kv = (unsigned)a.kv_heads;
    const long long rows = a.n * kv, step = (long long)gridDim.x * kRowWarps * HPW;
    for (long long r0 = ((long long)blockIdx.x * kRowWarps + (tid >> 5)) * HPW; r0 < rows; r0 += step) {
        const long long r = min(r0 + sub, rows - 1), tok = r / kv;
        const int h = (int)(r - tok * kv);
        const long long slot = a.slots[tok];
        const bool in = slot >= 0 && slot < a.num_slots;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        float as = 0.0f;
        if (in) {
            const size_t row = (((size_t)(slot >> a.page_shift) * kv + h) << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
            const uint32_t* wp = reinterpret_cast<const uint32_t*>(a.idx[side] + row * (D / 8 * BITS));
            uint32_t w;
            if (BITS == 4) {
                w = __ldg(wp + l);
            } else {
                const int k = (3 * l) >> 2;
                w = __funnelshift_r(__ldg(wp + k), __ldg(wp + min(k + 1, D * BITS / 32 - 1)), (24 * l) & 31);
            }
            as = fabsf(f16_bits_to_f32(__ldg(a.sc[side] + row * (D / 32) + (l >> 2))));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float c = s_tab[(w >> (BITS * i)) & (kCodes - 1)][lane];
                v[i] = ((neg >> i) & 1u) ? -c : c;
            }
        }
#pragma unroll
        for (int hh = 1; hh < 8; hh <<= 1)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((i & hh) == 0) {
                    const float x = v[i], y = v[i + hh];
                    v[i] = x + y;
                    v[i + hh] = x - y;
                }
#pragma unroll
        for (int m = 1; m <= 2; m <<= 1) {
            const bool upper = (lane & m) != 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float other = __shfl_xor_sync(0xffffffffu, v[i], m);
                v[i] = upper ? (other - v[i]) : (v[i] + other);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = in ? (v[i] * inv_sqrt) * as : 0.0f;
        if (r0 + sub < rows) {
            Eight<T> e;
            e.set(v);
            e.store(reinterpret_cast<T*>(a.out[side]) + r * D + 8 * l);
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
int log2_of(int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

size_t size_of(int dtype) { return dtype == TQB_F32 ? 4 : dtype == TQB_F16 || dtype == TQB_BF16 ? 2 : 0; }

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// Rows of `elem` bytes an element: dense heads of 16-byte pieces at non-negative strides.
int check_rows(const void* p, long long token, long long head, size_t elem) {
    if (token < 0 || head < 0) return TQB_ERR_INVALID_ARGUMENT;
    if (!aligned16(p) || (token * (long long)elem) % 16 != 0 || (head * (long long)elem) % 16 != 0) return TQB_ERR_MISALIGNED;
    return TQB_OK;
}

template <typename T, int LPH>
int launch_rows_bits(int bits, const RowArgs& a, const Codebook& cb, cudaStream_t s) {
    const int grid = a.tokens < 148 * 8 ? a.tokens : 148 * 8;
    switch (bits) {
        case 0: rows_kernel<T, LPH, 0><<<grid, kRowThreads, 0, s>>>(a, cb); break;
        case 3: rows_kernel<T, LPH, 3><<<grid, kRowThreads, 0, s>>>(a, cb); break;
        default: rows_kernel<T, LPH, 4><<<grid, kRowThreads, 0, s>>>(a, cb); break;
    }
    return check_launch(s);
}
template <typename T>
int launch_rows_dim(int dim, int bits, const RowArgs& a, const Codebook& cb, cudaStream_t s) {
    if (dim == 64) return launch_rows_bits<T, 8>(bits, a, cb, s);
    if (dim == 128) return launch_rows_bits<T, 16>(bits, a, cb, s);
    return launch_rows_bits<T, 32>(bits, a, cb, s);
}
int launch_rows(int dtype, int dim, int bits, RowArgs& a, cudaStream_t s) {
    Codebook cb{};
    if (bits != 0) {
        if (!block_codebook(bits, TQB_MAXNORM, cb)) return TQB_ERR_UNSUPPORTED_BITS;
        a.outer_centroid = cb.c[cb.n - 1];
    }
    if (dtype == TQB_F32) return launch_rows_dim<float>(dim, bits, a, cb, s);
    if (dtype == TQB_F16) return launch_rows_dim<__half>(dim, bits, a, cb, s);
    return launch_rows_dim<__nv_bfloat16>(dim, bits, a, cb, s);
}

int rope_args(const tqb_rope_params* p, bool keys_out, RowArgs& a) {
    if (!p) return TQB_ERR_NULL_POINTER;
    const size_t elem = size_of(p->dtype);
    if (elem == 0) return TQB_ERR_INVALID_ARGUMENT;
    if (p->head_dim <= 0 || p->head_dim % kBlock != 0) return TQB_ERR_INVALID_DIMENSION;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return TQB_ERR_UNSUPPORTED;
    if (p->rot_dim < 0 || p->rot_dim > p->head_dim || p->rot_dim % 16 != 0) return TQB_ERR_INVALID_ARGUMENT;
    if (p->num_tokens < 0 || p->num_q_heads < 0 || p->num_kv_heads < 0 || !(p->eps >= 0.0f)) return TQB_ERR_INVALID_ARGUMENT;
    if ((p->flags & ~(TQB_ROPE_INTERLEAVED | TQB_ROPE_NO_NORM | TQB_ROPE_POSITIONS_64)) != 0) return TQB_ERR_INVALID_ARGUMENT;
    if (p->num_tokens == 0) return TQB_OK;
    if (p->q && !p->q_out) return TQB_ERR_NULL_POINTER;
    if (p->k && keys_out && !p->k_out) return TQB_ERR_NULL_POINTER;
    if (p->rot_dim > 0) {
        if (!p->positions || !p->inv_freq) return TQB_ERR_NULL_POINTER;
        if ((uintptr_t)p->positions % ((p->flags & TQB_ROPE_POSITIONS_64) ? 8 : 4) != 0 || (uintptr_t)p->inv_freq % 4 != 0) return TQB_ERR_MISALIGNED;
    }
    int st = TQB_OK;
    if (p->q) {
        if ((st = check_rows(p->q, p->q_token_stride, p->q_head_stride, elem)) != TQB_OK) return st;
        if ((st = check_rows(p->q_out, p->q_out_token_stride, p->q_out_head_stride, elem)) != TQB_OK) return st;
        if (!aligned16(p->q_weight)) return TQB_ERR_MISALIGNED;
        a.q = RowSpan{p->q, p->q_out, p->q_token_stride, p->q_head_stride, p->q_out_token_stride, p->q_out_head_stride, p->q_weight, p->num_q_heads};
    }
    if (p->k) {
        if ((st = check_rows(p->k, p->k_token_stride, p->k_head_stride, elem)) != TQB_OK) return st;
        if (p->k_out && (st = check_rows(p->k_out, p->k_out_token_stride, p->k_out_head_stride, elem)) != TQB_OK) return st;
        if (!aligned16(p->k_weight)) return TQB_ERR_MISALIGNED;
        a.k = RowSpan{p->k, p->k_out, p->k_token_stride, p->k_head_stride, p->k_out_token_stride, p->k_out_head_stride, p->k_weight, p->num_kv_heads};
    }
    a.positions = p->positions;
    a.inv_freq = p->inv_freq;
    a.tokens = p->num_tokens;
    a.rot_dim = p->rot_dim;
    a.flags = p->flags;
    a.eps = p->eps;
    return TQB_OK;
}

int layer_args(const tqb_paged_layer* l, const int64_t* slots, RowArgs& a) {
    if (!slots) return TQB_ERR_NULL_POINTER;
    if ((uintptr_t)slots % 8 != 0) return TQB_ERR_MISALIGNED;
    a.slots = slots;
    a.idx[0] = l->k_indices;
    a.idx[1] = l->v_indices;
    a.sc[0] = l->k_scales;
    a.sc[1] = l->v_scales;
    a.num_slots = (long long)l->num_pages * l->page_size;
    a.kv_heads = l->num_kv_heads;
    a.page_shift = log2_of(l->page_size);
    return TQB_OK;
}

int check_plan_shape(int32_t num_requests, int64_t table_stride, int32_t max_blocks, int32_t page_size) {
    if (num_requests < 0 || max_blocks < 0 || table_stride < max_blocks) return TQB_ERR_INVALID_ARGUMENT;
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0) return TQB_ERR_INVALID_ARGUMENT;
    if (num_requests > TQB_PAGED_MAX_REQUESTS) return TQB_ERR_TOO_LARGE;
    return TQB_OK;
}

}  // namespace

int check_paged_layer(const tqb_paged_layer* l) {
    if (!l) return TQB_ERR_NULL_POINTER;
    if (l->bits < 3 || l->bits > 4) return TQB_ERR_UNSUPPORTED_BITS;
    if (l->head_dim <= 0 || l->head_dim % kBlock != 0) return TQB_ERR_INVALID_DIMENSION;
    if (l->head_dim != 64 && l->head_dim != 128 && l->head_dim != 256) return TQB_ERR_UNSUPPORTED;
    if (l->page_size < 16 || l->page_size > 1024 || (l->page_size & (l->page_size - 1)) != 0) return TQB_ERR_INVALID_ARGUMENT;
    if (l->num_pages < 0 || l->num_kv_heads <= 0) return TQB_ERR_INVALID_ARGUMENT;
    // rows are counted in 32 bits: 2^32 rows of the smallest kind are 206 GB
    if ((unsigned long long)l->num_pages * l->num_kv_heads > (1ull << 32) / l->page_size - 1) return TQB_ERR_TOO_LARGE;
    if (l->num_pages == 0) return TQB_OK;
    if (!l->k_indices || !l->k_scales || !l->v_indices || !l->v_scales) return TQB_ERR_NULL_POINTER;
    if (!aligned16(l->k_indices) || !aligned16(l->k_scales) || !aligned16(l->v_indices) || !aligned16(l->v_scales)) return TQB_ERR_MISALIGNED;
    return TQB_OK;
}

}  // namespace tqb

using namespace tqb;

extern "C" {

int tqb_paged_plan(const int32_t* seq_lens, const int32_t* new_tokens, int32_t num_requests, int32_t* block_table,
                   int64_t table_stride, int32_t max_blocks, const int32_t* free_pages, int32_t* state, int32_t page_size,
                   int64_t* slots, int32_t* positions, int32_t capacity, int32_t* cu, int32_t* kv_lens, int32_t* state_out,
                   tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    int st = check_plan_shape(num_requests, table_stride, max_blocks, page_size);
    if (st != TQB_OK) return st;
    if (capacity < 0) return TQB_ERR_INVALID_ARGUMENT;
    if (!state || !state_out || !cu) return TQB_ERR_NULL_POINTER;
    if (num_requests > 0 && (!seq_lens || !new_tokens || !kv_lens || (max_blocks > 0 && (!block_table || !free_pages)))) return TQB_ERR_NULL_POINTER;
    if (capacity > 0 && (!slots || !positions)) return TQB_ERR_NULL_POINTER;
    PlanArgs a{seq_lens, new_tokens, block_table, table_stride, free_pages, state, slots, positions, cu, kv_lens, state_out,
               num_requests, max_blocks, log2_of(page_size), capacity};
    int grid = (capacity + kPlanTokens - 1) / kPlanTokens;
    grid = grid < 1 ? 1 : grid > 148 ? 148 : grid;
    plan_kernel<<<grid, kPlanThreads, 0, as_stream(stream)>>>(a);
    return check_launch(as_stream(stream));
}

int tqb_paged_release(const uint8_t* mask, int32_t* seq_lens, int32_t num_requests, int32_t* block_table, int64_t table_stride,
                      int32_t max_blocks, int32_t* free_pages, int32_t free_capacity, int32_t* state, int32_t page_size,
                      tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    int st = check_plan_shape(num_requests, table_stride, max_blocks, page_size);
    if (st != TQB_OK) return st;
    if (free_capacity < 0) return TQB_ERR_INVALID_ARGUMENT;
    if (!state) return TQB_ERR_NULL_POINTER;
    if (num_requests > 0 && (!mask || !seq_lens || (max_blocks > 0 && (!block_table || !free_pages)))) return TQB_ERR_NULL_POINTER;
    release_kernel<<<1, kReleaseThreads, 0, as_stream(stream)>>>(mask, seq_lens, num_requests, block_table, table_stride, max_blocks,
                                                                free_pages, free_capacity, state, log2_of(page_size));
    return check_launch(as_stream(stream));
}

int tqb_qk_norm_rope(const tqb_rope_params* p, tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    RowArgs a{};
    int st = rope_args(p, true, a);
    if (st != TQB_OK) return st;
    if (a.tokens == 0 || a.q.heads + a.k.heads == 0) return TQB_OK;
    return launch_rows(p->dtype, p->head_dim, 0, a, as_stream(stream));
}

int tqb_paged_append(const tqb_paged_layer* layer, const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                     int64_t v_token_stride, int64_t v_head_stride, int32_t dtype, const int64_t* slots, int32_t num_tokens,
                     tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    int st = check_paged_layer(layer);
    if (st != TQB_OK) return st;
    const size_t elem = size_of(dtype);
    if (elem == 0 || num_tokens < 0) return TQB_ERR_INVALID_ARGUMENT;
    if (num_tokens == 0 || layer->num_pages == 0) return TQB_OK;
    if (!k || !v) return TQB_ERR_NULL_POINTER;
    if ((st = check_rows(k, k_token_stride, k_head_stride, elem)) != TQB_OK) return st;
    if ((st = check_rows(v, v_token_stride, v_head_stride, elem)) != TQB_OK) return st;
    RowArgs a{};
    if ((st = layer_args(layer, slots, a)) != TQB_OK) return st;
    a.k = RowSpan{k, nullptr, k_token_stride, k_head_stride, 0, 0, nullptr, layer->num_kv_heads};
    a.v = RowSpan{v, nullptr, v_token_stride, v_head_stride, 0, 0, nullptr, layer->num_kv_heads};
    a.tokens = num_tokens;
    a.flags = TQB_ROPE_NO_NORM;
    return launch_rows(dtype, layer->head_dim, layer->bits, a, as_stream(stream));
}

int tqb_paged_append_rope(const tqb_paged_layer* layer, const tqb_rope_params* p, const void* v, int64_t v_token_stride,
                          int64_t v_head_stride, const int64_t* slots, tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    int st = check_paged_layer(layer);
    if (st != TQB_OK) return st;
    RowArgs a{};
    if ((st = rope_args(p, false, a)) != TQB_OK) return st;
    if (p->head_dim != layer->head_dim || p->num_kv_heads != layer->num_kv_heads) return TQB_ERR_DIMENSION_MISMATCH;
    if (a.tokens == 0) return TQB_OK;
    if (!p->k || !v) return TQB_ERR_NULL_POINTER;
    if ((st = check_rows(v, v_token_stride, v_head_stride, size_of(p->dtype))) != TQB_OK) return st;
    if ((st = layer_args(layer, slots, a)) != TQB_OK) return st;
    a.v = RowSpan{v, nullptr, v_token_stride, v_head_stride, 0, 0, nullptr, layer->num_kv_heads};
    return launch_rows(p->dtype, p->head_dim, layer->bits, a, as_stream(stream));
}

int tqb_paged_dequantize(const tqb_paged_layer* layer, const int64_t* slots, int64_t n, void* k_out, void* v_out, int32_t out_dtype,
                         tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    int st = check_paged_layer(layer);
    if (st != TQB_OK) return st;
    if (n < 0 || size_of(out_dtype) == 0) return TQB_ERR_INVALID_ARGUMENT;
    if (n == 0) return TQB_OK;
    if (!slots || !k_out || !v_out) return TQB_ERR_NULL_POINTER;
    if ((uintptr_t)slots % 8 != 0 || !aligned16(k_out) || !aligned16(v_out)) return TQB_ERR_MISALIGNED;
    BackArgs a{{layer->k_indices, layer->v_indices}, {layer->k_scales, layer->v_scales}, {k_out, v_out}, slots, n,
               (long long)layer->num_pages * layer->page_size, layer->num_kv_heads, log2_of(layer->page_size), block_sign_magnitude()};
    Codebook cb{};
    if (!block_codebook(layer->bits, TQB_MAXNORM, cb)) return TQB_ERR_UNSUPPORTED_BITS;
    const int lph = layer->head_dim / 8;
    const long long warps = (n * layer->num_kv_heads * lph + 31) / 32, want = (warps + kRowWarps - 1) / kRowWarps;
    const dim3 grid((unsigned)(want < 148 * 8 ? want : 148 * 8), 2);
    cudaStream_t s = as_stream(stream);
#define TQB_BACK(T, LPH)                                                               \
    do {                                                                               \
        if (layer->bits == 3) back_kernel<T, LPH, 3><<<grid, kRowThreads, 0, s>>>(a, cb); \
        else back_kernel<T, LPH, 4><<<grid, kRowThreads, 0, s>>>(a, cb);               \
    } while (0)
#define TQB_BACK_DIM(T)                 \
    do {                                \
        if (lph == 8) TQB_BACK(T, 8);   \
        else if (lph == 16) TQB_BACK(T, 16); \
        else TQB_BACK(T, 32);           \
    } while (0)
    if (out_dtype == TQB_F32) TQB_BACK_DIM(float);
    else if (out_dtype == TQB_F16) TQB_BACK_DIM(__half);
    else TQB_BACK_DIM(__nv_bfloat16);
#undef TQB_BACK_DIM
#undef TQB_BACK
    return check_launch(s);
}

}  // extern "C"
