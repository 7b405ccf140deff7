// How the kernels of the paged attention share their work, and how the shares are joined.
//
// The work of a call is a line of tiles of kTile tokens: request after request, within a request KV head after KV head
// (a group of more than eight query heads counts as several), within a head token after token.  CTA i of n takes the tiles
// [i W / n, (i + 1) W / n): equal shares whatever the lengths are, worked out on the device from the lengths, so that a
// captured launch serves any batch.  A share is cut into segments, one for each (request, head) that it touches.  A segment
// that is the whole of its (request, head) is written to the output; otherwise its sum, maximum and un-normalised output go
// to the scratch (a CTA has at most two such segments: its first and its last), and the CTA that arrives last at the
// (request, head)'s ticket joins them in the order of the CTAs.  The result depends on the lengths alone.
#pragma once
#include "tqb_common.cuh"
#include "tqb_paged.cuh"

namespace tqb {

constexpr int kTile = 64;            // tokens
constexpr int kSegHeads = 8;         // query heads of a segment, at most
constexpr int kWorkThreads = 128;
constexpr int kMaxCtas = 148 * 8;    // of a launch: sizes tickets and partials
static_assert(kMaxCtas * 4 <= TQB_PAGED_TICKET_BYTES, "a ticket for each CTA");
constexpr float kNoScore = -1.0e30f; // finite stand-in for -inf: differences of two of them are 0

struct PagedArgs {
    const void* q;
    void* out;
    const uint8_t* kb;
    const uint16_t* ks;
    const uint8_t* vb;
    const uint16_t* vs;
    const int32_t* table;
    const int32_t* lens;
    unsigned* tickets;
    float* part_ml;      // [kMaxCtas][2][kSegHeads][2]: maximum (log2 units), sum
    float* part_out;     // [kMaxCtas][2][kSegHeads][D], rotated domain
    long long q_stride, table_stride;
    int requests, max_blocks, page_shift, num_pages, hkv, group, vheads, splits;   // vheads = hkv * splits
    int q_dtype, out_dtype;
    float qk_const;      // softmax_scale * log2(e)
    float sign_mag;
    float cent[16];
};

int launch_paged_mma(const PagedArgs& a, int head_dim, cudaStream_t s);   // 4-bit, 16-bit queries, some page

struct Segment {
    int req, kvh, head0, heads;   // query heads head0 .. head0 + heads - 1 of the request
    int t0, t1;                   // its tokens
    bool whole;
    int first, parts;             // not whole: the first CTA of the (request, head), and how many there are
    int slot;                     // where this CTA's part goes: cta * 2 + (0: it began before this CTA, 1: it goes on behind it)
};

struct WorkLine {
    const PagedArgs& a;
    long long total, ctas, cur, end, base;   // tiles; base: first tile of request `req`
    int req, tiles, len;

    __device__ __forceinline__ int length(int r) const {
        const long long cap = min((long long)a.max_blocks << a.page_shift, 0x7fffffc0ll);
        return (int)min((long long)max(a.lens[r], 0), cap);
    }
    static __device__ __forceinline__ int tiles_of(int len) { return (len + kTile - 1) / kTile; }

    // All threads of the CTA.  Reads every request's length (4 bytes each, from L2): two block barriers.
    __device__ __forceinline__ explicit WorkLine(const PagedArgs& args) : a(args) {
        __shared__ long long s_sum[kWorkThreads / 32];
        __shared__ long long s_base;
        __shared__ int s_req;
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const int per = (a.requests + kWorkThreads - 1) / kWorkThreads, r0 = min(tid * per, a.requests), r1 = min(r0 + per, a.requests);
        long long mine = 0;
        for (int r = r0; r < r1; ++r) mine += tiles_of(length(r));
        long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        total = 0;
        long long before = incl - mine;
#pragma unroll
        for (int w = 0; w < kWorkThreads / 32; ++w) {
            if (w < warp) before += s_sum[w];
            total += s_sum[w];
        }
        total *= a.vheads;
        ctas = min((long long)gridDim.x, total);
        cur = end = base = 0;
        req = tiles = len = 0;
        if ((long long)blockIdx.x >= ctas) return;   // (the same for the whole CTA)
        cur = blockIdx.x * total / ctas;
        end = (blockIdx.x + 1) * total / ctas;
        const long long at = before * a.vheads;
        if (at <= cur && cur < at + mine * a.vheads) {
            long long b = at;
            int r = r0;
            for (; r < r1 - 1; ++r) {
                const long long n = (long long)tiles_of(length(r)) * a.vheads;
                if (cur < b + n) break;
                b += n;
            }
            s_req = r;
            s_base = b;
        }
        __syncthreads();
        req = s_req;
        base = s_base;
        len = length(req);
        tiles = tiles_of(len);
        if (tiles == 0) end = cur;
    }

    __device__ __forceinline__ bool more() const { return cur < end; }

    // The segment at `cur`; moves on behind it.
    __device__ __forceinline__ Segment next() {
        Segment s;
        const long long off = cur - base;
        const int vh = (int)(off / tiles), t = (int)(off - (long long)vh * tiles);
        const int n = (int)min((long long)(tiles - t), end - cur);
        s.req = req;
        s.kvh = vh / a.splits;
        const int g0 = (vh - s.kvh * a.splits) * kSegHeads;
        s.head0 = s.kvh * a.group + g0;
        s.heads = min(a.group - g0, kSegHeads);
        s.t0 = t * kTile;
        s.t1 = min((t + n) * kTile, len);
        s.whole = n == tiles;
        s.first = 0;
        s.parts = 1;
        s.slot = blockIdx.x * 2 + (t == 0 ? 1 : 0);
        if (!s.whole) {   // tile x belongs to CTA floor(((x + 1) ctas - 1) / total)
            const long long x0 = cur - t, x1 = x0 + tiles - 1;
            s.first = (int)(((x0 + 1) * ctas - 1) / total);
            s.parts = (int)(((x1 + 1) * ctas - 1) / total) - s.first + 1;
        }
        cur += n;
        if (cur < end && cur == base + (long long)tiles * a.vheads) {
            base = cur;
            len = 0;
            while (len == 0 && req + 1 < a.requests) len = length(++req);
            tiles = tiles_of(len);
            if (tiles == 0) end = cur;   // not reached while the lengths stay as they are
        }
        return s;
    }
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float wht32_across(float v, int lane) {
#pragma unroll
    for (int h = 1; h < 32; h <<= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, v, h);
        v = (lane & h) ? (other - v) : (v + other);
    }
    return v;
}

__device__ __forceinline__ float block_sign(int lane, float mag) {   // src/cache/precomputed/rotation.rs:16-20
    return ((0xB1A6D4B2u >> lane) & 1u) ? -mag : mag;
}

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, size_t i) {
    if (dtype == TQB_F32) return reinterpret_cast<const float*>(p)[i];
    if (dtype == TQB_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_as(void* p, int dtype, size_t i, float v) {
    if (dtype == TQB_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (dtype == TQB_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Rotated sum O over the softmax sum L of (head, block b), one lane a dim, back through the rotation and out.
template <int NB>
__device__ __forceinline__ void write_block(const PagedArgs& a, const Segment& s, int hh, int b, int lane, float O, float L) {
    const float r = wht32_across(O * block_sign(lane, a.sign_mag), lane) * (1.0f / sqrtf((float)kBlock));
    // L is 0 where no page of the request can be read
    store_as(a.out, a.out_dtype, ((size_t)s.req * a.hkv * a.group + s.head0 + hh) * (NB * 32) + b * 32 + lane, L == 0.0f ? 0.0f : r / L);
}

// The segment's end, by all threads of the CTA: `value(warp, head, dim)` is a warp's un-normalised rotated output relative to
// its maximum s_m[warp][head], s_l its sum.  A (head, block) unit a warp at a time.
template <int NB, typename F>
__device__ __forceinline__ void finish_segment(const PagedArgs& a, const Segment& s, const float (*s_m)[kSegHeads], const float (*s_l)[kSegHeads], F value) {
    constexpr int kWarps = kWorkThreads / 32, D = NB * 32;
    __shared__ int s_arrived;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int u = warp; u < s.heads * NB; u += kWarps) {
        const int hh = u / NB, b = u - hh * NB;
        float M = s_m[0][hh];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w][hh]);
        float L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float e = exp2_fast(s_m[w][hh] - M);
            L = fmaf(s_l[w][hh], e, L);
            O = fmaf(value(w, hh, b * 32 + lane), e, O);
        }
        if (s.whole) {
            write_block<NB>(a, s, hh, b, lane, O, L);
        } else {
            const size_t at = (size_t)s.slot * kSegHeads + hh;
            a.part_out[at * D + b * 32 + lane] = O;
            if (b == 0 && lane == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(M, L);
        }
    }
    if (s.whole) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_arrived = atomicAdd(a.tickets + s.first, 1u) == (unsigned)(s.parts - 1);
    __syncthreads();
    if (!s_arrived) return;
    __threadfence();
    for (int u = warp; u < s.heads * NB; u += kWarps) {
        const int hh = u / NB, b = u - hh * NB;
        // part 0 is the second slot of CTA `first`, part i the first slot of CTA first + i
        auto at = [&](int i) { return (size_t)((s.first + i) * 2 + (i == 0 ? 1 : 0)) * kSegHeads + hh; };
        float M = kNoScore;
        for (int i = lane; i < s.parts; i += 32) M = fmaxf(M, __ldcg(a.part_ml + at(i) * 2));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        float L = 0.0f, O = 0.0f;
        for (int i0 = 0; i0 < s.parts; i0 += 32) {
            float w = 0.0f;
            if (i0 + lane < s.parts) {
                const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml + at(i0 + lane) * 2));
                w = exp2_fast(ml.x - M);
                L = fmaf(ml.y, w, L);
            }
            const int n = min(32, s.parts - i0);
            for (int i = 0; i < n; i += 8) {
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = i + k < n ? __ldcg(a.part_out + at(i0 + i + k) * D + b * 32 + lane) : 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) O = fmaf(v[k], __shfl_sync(0xffffffffu, w, (i + k) & 31), O);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        write_block<NB>(a, s, hh, b, lane, O, L);
    }
    __syncthreads();
    if (threadIdx.x == 0) a.tickets[s.first] = 0u;   // ready for the next call
}

// Requests without tokens get zeros.
template <int NB>
__device__ __forceinline__ void write_empty(const PagedArgs& a) {
    const int row = a.hkv * a.group * NB * 32;
    for (int r = blockIdx.x; r < a.requests; r += gridDim.x) {
        if (a.lens[r] > 0 && a.max_blocks > 0) continue;
        for (int i = threadIdx.x; i < row; i += kWorkThreads) store_as(a.out, a.out_dtype, (size_t)r * row + i, 0.0f);
    }
}

}  // namespace tqb
