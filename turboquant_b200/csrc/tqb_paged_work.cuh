// How the kernels of the paged attention share their work, and how the shares are joined.
//
// The work of a call is a line of units: groups of 16 tokens (16 << unit_shift, where 2^30 units could not count the widest
// table), request after request, within a request KV head after KV head (a group of more than eight query heads counts as
// several), within a head token after token; kOpenCost units stand before each (request, head) for what it takes to begin
// one.  Every WARP takes an equal run of the line, whatever the lengths are, worked out on the device from the lengths, so
// that a captured launch serves any batch.  A run is cut into segments, one for each (request, head) that it touches.  A warp
// writes a segment that is the whole of its (request, head) to the output by itself.  It has at most two others: one that began
// before it and one that goes on behind it.  These stay in shared memory until the CTA's four warps are done and are joined
// there, and what crosses the CTA's ends goes to the scratch (again at most two parts), where the CTA that arrives last at the
// (request, head)'s ticket joins the parts in the order of the CTAs.  How the sums are cut and ordered depends on the lengths and on
// the call's shape (heads, number of requests, width of the table), so that a call repeats bit for bit.
//
// Measured at 128 requests of 62 to 1,000 tokens (8 KV heads, 4-bit): with CTAs instead of warps taking the runs, every
// short segment paid its loads' latency and eight block barriers: 64 us.
#pragma once
#include <float.h>

#include "tqb_common.cuh"
#include "tqb_mma.cuh"
#include "tqb_paged.cuh"

namespace tqb {

constexpr int kRunTokens = 16;       // of a group
// Measured with 3, 4, 5, 6, 8 groups: 64 requests of 531 to 8,192 tokens 44.6, 44.7, 44.3, 43.8, 43.9 us, 256 of 19 to 300 tokens
// 21.9, 20.9, 20.6, 21.0, 21.1; and with runs of at least 2, 4, 6, 8 units: one request of 1,000 tokens 9.3, 10.3, 10.0, 10.7, four of
// them 11.0, 10.3, 10.0, 10.7.
constexpr int kOpenCost = 6;         // groups that beginning a segment is worth
constexpr int kMinRun = 6;           // units of a run, at least
constexpr int kSegHeads = 8;         // query heads of a segment, at most
constexpr int kWorkWarps = 4;
constexpr int kWorkThreads = 32 * kWorkWarps;
constexpr int kMaxCtas = 148 * 8;    // of a launch: sizes tickets and partials
constexpr int kMaxRound = 36;        // parts joined at a time, at most
static_assert(kMaxCtas * 3 * 4 <= TQB_PAGED_TICKET_BYTES, "tickets of the last round, and of the slots for the one before it");
constexpr float kNoScore = -FLT_MAX; // finite stand-in for -inf: differences of two of them are 0

struct PagedArgs {
    const void* q;
    void* out;
    const uint8_t* kb;
    const uint16_t* ks;
    const uint8_t* vb;
    const uint16_t* vs;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu;   // [requests + 1] first token of each request in the step whose tokens are the rows of q and out, or nullptr: row r is request r
    unsigned* tickets;
    float* part_ml;      // [kMaxCtas][2][kSegHeads][2]: maximum (log2 units), sum
    float* round_ml;     // the same of joined parts, where two rounds are needed
    float* part_out;     // [kMaxCtas][2][kSegHeads][D], rotated domain
    long long q_stride, table_stride;
    int requests, rows, max_blocks, max_len, unit_shift, page_shift, num_pages, hkv, group, vheads, splits;   // vheads = hkv * splits
    int q_dtype, out_dtype;
    float qk_const;      // softmax_scale * log2(e)
    float sign_mag;
    float cent[16];
    // 3-bit, tensor-core kernel: centroid / kappa, and centroids / the largest * 32639 in two base-256 digits ([0..1] the high ones)
    float kappa, values[8];
    uint32_t digits[4];
};

int launch_paged_mma(const PagedArgs& a, int head_dim, int bits, cudaStream_t s);   // 16-bit queries, some page

// The row of request r, or -1 where it has none: among the tokens of a step a request that brings exactly one has that one.
__device__ __forceinline__ int row_of(const PagedArgs& a, int r) {
    if (a.cu == nullptr) return r;
    const int row = a.cu[r];
    return (unsigned)a.cu[r + 1] - (unsigned)row == 1u && (unsigned)row < (unsigned)a.rows ? row : -1;
}
__device__ __forceinline__ int known_row(const PagedArgs& a, int r) { return a.cu == nullptr ? r : a.cu[r]; }   // of a request that has one

struct Segment {
    int req, kvh, head0, heads;   // query heads head0 .. head0 + heads - 1 of the request
    int t0, t1;                   // its tokens
    bool begins, ends;            // it has the first, the last token of its (request, head)
    int cta0, ctas;               // the CTAs that share the (request, head)
    __device__ __forceinline__ bool whole() const { return begins && ends; }
};

// x / y for quotients below 2^21: the f32 quotient (x, y rounded to 2^-24, __fdividef good to 2 ulp: 2^-21.4 in all) is then off
// by less than 1, so one step mends it.  (An integer
// division is some 50 instructions one behind the other, and a run begins with seven of them.)
__device__ __forceinline__ unsigned divide(unsigned x, unsigned y) {
    unsigned q = (unsigned)__fdividef((float)x, (float)y);
    const int r = (int)(x - q * y);
    q += r < 0 ? -1 : r >= (int)y ? 1 : 0;
    return q;
}

// A warp's run of the line.
struct WorkLine {
    const PagedArgs& a;
    unsigned quot, rem;              // a run has quot units, the first `rem` runs one more
    unsigned cur, end, base;         // base: where request `req` begins
    int req, len;

    __device__ __forceinline__ int length(int r) const { return row_of(a, r) < 0 ? 0 : min(max(a.lens[r], 0), a.max_len); }
    __device__ __forceinline__ unsigned groups_of(int l) const { return ((unsigned)l + (kRunTokens << a.unit_shift) - 1) / kRunTokens >> a.unit_shift; }
    __device__ __forceinline__ unsigned units_of(int l) const { return l > 0 ? kOpenCost + groups_of(l) : 0u; }
    __device__ __forceinline__ int owner(unsigned x) const {   // the run that unit x belongs to
        const unsigned split = rem * (quot + 1);
        return (int)(x < split ? divide(x, quot + 1) : rem + divide(x - split, quot));
    }

    // All threads of the CTA.  Reads every request's length (4 bytes each, from L2): two block barriers.
    __device__ __forceinline__ explicit WorkLine(const PagedArgs& args) : a(args) {
        __shared__ unsigned s_sum[kWorkWarps], s_begin[kWorkThreads];
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const int per = (a.requests + kWorkThreads - 1) / kWorkThreads, r0 = min(tid * per, a.requests), r1 = min(r0 + per, a.requests);
        unsigned mine = 0;
#pragma unroll 1
        for (int r = r0; r < r1; ++r) mine += units_of(length(r));
        unsigned incl = mine;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        unsigned total = 0, before = incl - mine;
#pragma unroll
        for (int w = 0; w < kWorkWarps; ++w) {
            if (w < warp) before += s_sum[w];
            total += s_sum[w];
        }
        s_begin[tid] = before * a.vheads;
        __syncthreads();
        total *= a.vheads;
        // as many runs as the longest run needs: it is no longer with them, and fewer parts are joined
        const unsigned most = gridDim.x * kWorkWarps, i = blockIdx.x * kWorkWarps + warp;
        const unsigned longest = max(divide(total + most - 1, most), min(total, (unsigned)kMinRun));
        const unsigned runs = longest > 0 ? divide(total + longest - 1, longest) : 0;
        cur = end = base = 0;
        quot = rem = 0;
        req = len = 0;
        if (i >= runs) return;
        quot = divide(total, runs);
        rem = total - quot * runs;
        cur = i * quot + min(i, rem);
        end = cur + quot + (i < rem ? 1 : 0);
        // the last of the threads' requests that begin at or before `cur`: four threads a lane, then their requests
        int chunk = 0;
#pragma unroll
        for (int k = 0; k < kWorkWarps; ++k) chunk += __popc(__ballot_sync(0xffffffffu, s_begin[32 * k + lane] <= cur));
        --chunk;   // (threads behind the last request begin at the total)
        base = s_begin[chunk];
        req = min(chunk * per, a.requests - 1);
        len = length(req);
        while (req + 1 < a.requests && cur >= base + units_of(len) * a.vheads) {
            base += units_of(len) * a.vheads;
            len = length(++req);
        }
        if (len == 0) end = cur;   // not reached while the lengths stay as they are
    }

    // The next segment; false at the run's end.
    __device__ __forceinline__ bool next(Segment& s) {
        while (cur < end) {
            const unsigned groups = groups_of(len), units = kOpenCost + groups, vh = divide(cur - base, units), start = base + vh * units;
            const unsigned u0 = cur - start, u1 = min(units, u0 + (end - cur));
            const unsigned g0 = max(u0, (unsigned)kOpenCost) - kOpenCost, g1 = max(u1, (unsigned)kOpenCost) - kOpenCost;
            s.req = req;
            s.kvh = a.splits == 1 ? (int)vh : (int)vh / a.splits;
            const int h0 = ((int)vh - s.kvh * a.splits) * kSegHeads;
            s.head0 = s.kvh * a.group + h0;
            s.heads = min(a.group - h0, kSegHeads);
            s.t0 = (int)(g0 << a.unit_shift) * kRunTokens;
            s.t1 = g1 == groups ? len : (int)(g1 << a.unit_shift) * kRunTokens;
            s.begins = g0 == 0;
            s.ends = g1 == groups;
            s.cta0 = s.ctas = 0;
            if (!s.whole()) {
                s.cta0 = owner(start + kOpenCost) / kWorkWarps;
                s.ctas = owner(start + units - 1) / kWorkWarps - s.cta0 + 1;
            }
            cur += u1 - u0;
            if (cur < end && cur == base + units * a.vheads) {
                base = cur;
                len = 0;
                while (len == 0 && req + 1 < a.requests) len = length(++req);
                if (len == 0) end = cur;   // not reached while the lengths stay as they are
            }
            if (g1 > g0) return true;
        }
        return false;
    }
};

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

__device__ __forceinline__ void store4(void* p, int dtype, size_t i, const float (&v)[4]) {   // i: a multiple of 4
    if (dtype == TQB_F32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (dtype == TQB_F16) {
        const __half2 x = __floats2half2_rn(v[0], v[1]), y = __floats2half2_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p) + i) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    } else {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v[0], v[1]), y = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p) + i) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    }
}

// Outputs leave four dims a lane, lane l of a warp with dims 4 (l modulo 8) .. of a 32-block: the rotated output O over the
// softmax sum L, back through the rotation (stages 1, 2 in the lane, 4, 8, 16 between lanes), to elements i .. i + 3.  All
// lanes of the warp take part.  Not inlined, like what else runs once a segment: code that runs once waits for its
// instructions more than for anything else (10 of 18 stalls an instruction in a call of one short request).
static __device__ __noinline__ void write_quad(void* out, int dtype, size_t i, bool live, float4 O, float L, float sign_mag) {
    const int lane = threadIdx.x & 31;
    const uint32_t neg = 0xB1A6D4B2u >> (4 * (lane & 7));   // src/cache/precomputed/rotation.rs:16-20
    float v[4] = {(neg & 1u) ? -O.x : O.x, (neg & 2u) ? -O.y : O.y, (neg & 4u) ? -O.z : O.z, (neg & 8u) ? -O.w : O.w};
    const float p = v[0] + v[1], q = v[0] - v[1], r = v[2] + v[3], t = v[2] - v[3];
    v[0] = p + r;
    v[1] = q + t;
    v[2] = p - r;
    v[3] = q - t;
#pragma unroll 1
    for (int m = 1; m <= 4; m <<= 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float other = __shfl_xor_sync(0xffffffffu, v[k], m);
            v[k] = (lane & m) ? (other - v[k]) : (v[k] + other);
        }
    const float inv = L == 0.0f ? 0.0f : __fdividef(sign_mag * (1.0f / sqrtf((float)kBlock)), L);   // L is 0 where no page of the request can be read
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= inv;
    if (live) store4(out, dtype, i, v);
}
template <int NB>
__device__ __forceinline__ size_t quad_at(const PagedArgs& a, const Segment& s, int x) {   // element 4 x of the segment's heads
    return ((size_t)known_row(a, s.req) * a.hkv * a.group + s.head0) * (NB * 32) + 4 * x;
}

// How many of a (request, head)'s parts are joined at a time: up to 24 at once, more of them in two rounds.  (A round is a
// fence, a ticket and two dependent trips to L2, about 2.5 us; 93 parts in one round took a CTA 30 us.)
__device__ __forceinline__ int parts_per_round(int parts) { return parts <= 24 ? parts : parts <= 64 ? 8 : parts <= 256 ? 16 : kMaxRound; }
static_assert(kMaxRound * kMaxRound >= kMaxCtas, "two rounds are enough");

// Where part i of a (request, head) lies: of the first CTA the second slot, of the others the first.
__device__ __forceinline__ unsigned part_at(int cta0, int i) { return (unsigned)((cta0 + i) * 2 + (i == 0 ? 1 : 0)) * kSegHeads; }

// A running (maximum, sum, output) of a softmax, four dims of a head.
struct Running {
    float M = kNoScore, L = 0.0f;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __device__ __forceinline__ void raise(float m) {
        const float to = fmaxf(M, m), keep = ex2(M - to);
        M = to;
        L *= keep;
        O.x *= keep;
        O.y *= keep;
        O.z *= keep;
        O.w *= keep;
    }
    __device__ __forceinline__ void add(float m, float l, float4 o) {   // m is not above M
        const float e = ex2(m - M);
        L = fmaf(l, e, L);
        O.x = fmaf(o.x, e, O.x);
        O.y = fmaf(o.y, e, O.y);
        O.z = fmaf(o.z, e, O.z);
        O.w = fmaf(o.w, e, O.w);
    }
};

// Parts i0, i0 + stride, .. (`count` of them) of a (request, head) that a CTA has to join: into the output, or (first: the first
// of two rounds) into the place of part i0, with maximum and sum in a place of their own, since other threads still read
// part i0's.
struct Join {
    int count, i0, stride, first;
};

// Every thread reads the maxima and sums of its head for itself, beside the outputs: one trip to L2 for kAtOnce parts, no
// barrier.
template <int NB>
__device__ __forceinline__ void join_parts(const PagedArgs& a, const Segment& s, const Join& j) {
    constexpr int D = NB * 32, kAtOnce = 4;
    const int lane = threadIdx.x & 31, quads = s.heads * (D / 4);
#pragma unroll 1
    for (int x0 = (int)threadIdx.x - lane; x0 < quads; x0 += kWorkThreads) {
        const int x = min(x0 + lane, quads - 1), hh = x / (D / 4);
        const float2* ml_in = reinterpret_cast<const float2*>(j.stride > 1 ? a.round_ml : a.part_ml) + hh;
        const float4* out_in = reinterpret_cast<const float4*>(a.part_out) + x;
        Running r;
#pragma unroll 1
        for (int i = 0; i < j.count; i += kAtOnce) {
            float4 v[kAtOnce];
            float2 ml[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {   // (past the end: the last part again, with weight 0)
                const unsigned at = part_at(s.cta0, j.i0 + min(i + k, j.count - 1) * j.stride);
                ml[k] = __ldcg(ml_in + at);
                v[k] = __ldcg(out_in + at * (D / 4));
            }
            float top = ml[0].x;
#pragma unroll
            for (int k = 1; k < kAtOnce; ++k) top = fmaxf(top, ml[k].x);
            r.raise(top);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k)
                if (i + k < j.count) r.add(ml[k].x, ml[k].y, v[k]);
        }
        const bool live = x0 + lane < quads;
        if (!j.first) {
            write_quad(a.out, a.out_dtype, quad_at<NB>(a, s, x), live, r.O, r.L, a.sign_mag);
        } else if (live) {
            const unsigned at = part_at(s.cta0, j.i0);
            reinterpret_cast<float4*>(a.part_out)[at * (D / 4) + x] = r.O;
            if (x % (D / 4) == 0) reinterpret_cast<float2*>(a.round_ml)[at + hh] = make_float2(r.M, r.L);
        }
    }
}

// A CTA's segments that are not whole: of each warp the one that began before it (slot 2 w) and the one that goes on behind it
// (slot 2 w + 1).  A segment that began before the warp and goes on behind it has slot 2 w.
struct Fragments {
    Segment seg[2 * kWorkWarps];
    float m[2 * kWorkWarps][kSegHeads], l[2 * kWorkWarps][kSegHeads];   // maximum (log2 units) and sum
    int used[2 * kWorkWarps];
};

// The CTA's end, by all of its threads: quad(slot, x) are four of a fragment's un-normalised rotated outputs.
template <int NB, typename F>
__device__ __forceinline__ void finish(const PagedArgs& a, const Fragments& f, F quad) {
    constexpr int D = NB * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    unsigned used = 0;
#pragma unroll
    for (int c = 0; c < 2 * kWorkWarps; ++c) used |= f.used[c] ? 1u << c : 0u;
    int crossing[2] = {-1, -1};   // a slot of the (request, head) that crosses the CTA's beginning | only its end
    while (used != 0) {
        const int c0 = __ffs(used) - 1;
        // the fragments of one (request, head): up to the next odd slot
        const unsigned odd = used & 0xaau & ~((2u << c0) - 1), mine = used & (odd != 0 ? (odd & (0u - odd)) - 1 : ~0u);
        used &= ~mine;
        const int last = 31 - __clz(mine), count = __popc(mine);
        const Segment& s = f.seg[c0];
        const bool done = s.begins && f.seg[last].ends;
        const int side = s.begins ? 1 : 0;
        if (!done) crossing[side] = c0;
        const int quads = s.heads * (D / 4);
        const size_t at = (size_t)(blockIdx.x * 2 + side) * kSegHeads;
#pragma unroll 1
        for (int x0 = warp * 32; x0 < quads; x0 += kWorkThreads) {
            const int x = min(x0 + lane, quads - 1), hh = x / (D / 4);
            // at most one fragment of a warp: read together (past the last: that one again, with weight 0)
            float m[kWorkWarps], l[kWorkWarps];
            float4 o[kWorkWarps];
            unsigned left = mine;
            int c = c0;
#pragma unroll
            for (int k = 0; k < kWorkWarps; ++k) {
                c = left != 0 ? __ffs(left) - 1 : c;
                left &= left - 1;
                m[k] = f.m[c][hh];
                l[k] = f.l[c][hh];
                o[k] = quad(c, x);
            }
            Running r;
#pragma unroll
            for (int k = 0; k < kWorkWarps; ++k) r.M = fmaxf(r.M, m[k]);
#pragma unroll
            for (int k = 0; k < kWorkWarps; ++k)
                if (k < count) r.add(m[k], l[k], o[k]);
            if (done) {
                write_quad(a.out, a.out_dtype, quad_at<NB>(a, s, x), x0 + lane < quads, r.O, r.L, a.sign_mag);
            } else if (x0 + lane < quads) {
                reinterpret_cast<float4*>(a.part_out + at * D)[x] = r.O;
                if (x % (D / 4) == 0) reinterpret_cast<float2*>(a.part_ml)[at + hh] = make_float2(r.M, r.L);
            }
        }
    }
    if (crossing[0] < 0 && crossing[1] < 0) return;
    // What crosses the CTA's ends: a first round of parts, if there are many, and the last one.  Warp 0 arrives for what crosses
    // the beginning, warp 1 for the rest, after everything that the CTA's threads have written; the last one to arrive sees
    // what the others have written and joins.
    __shared__ Join s_join[2];
#pragma unroll 1
    for (int round = 0; round < 2; ++round) {
        __syncthreads();
        if (lane == 0 && warp < 2) {
            const int c = warp == 0 ? crossing[0] : crossing[1];
            Join j{0, 0, 1, 0};
            if (c >= 0 && (round == 0 || s_join[warp].first)) {
                const int parts = f.seg[c].ctas, cta0 = f.seg[c].cta0, per = parts_per_round(parts);
                unsigned* ticket = a.tickets + cta0;
                int want = parts;
                if (per < parts && round == 0) {
                    j.i0 = ((int)blockIdx.x - cta0) / per * per;
                    j.first = 1;
                    want = min(per, parts - j.i0);
                    ticket = a.tickets + kMaxCtas + (cta0 + j.i0) * 2 + (j.i0 == 0 ? 1 : 0);
                } else if (per < parts) {
                    j.stride = per;
                    want = (parts + per - 1) / per;
                }
                unsigned old;
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;\n" : "=r"(old) : "l"(ticket) : "memory");
                if (old == (unsigned)(want - 1)) {
                    j.count = want;
                    *ticket = 0u;   // ready for the next call
                } else {
                    j.first = 0;
                }
            }
            s_join[warp] = j;
        }
        __syncthreads();
#pragma unroll 1
        for (int side = 0; side < 2; ++side)
            if (s_join[side].count > 0) join_parts<NB>(a, f.seg[side == 0 ? crossing[0] : crossing[1]], s_join[side]);
        if (!s_join[0].first && !s_join[1].first) return;
    }
}

// Requests without tokens get zeros; rows that no request has stay as they are.
template <int NB>
__device__ __forceinline__ void write_empty(const PagedArgs& a) {
    const int row = a.hkv * a.group * NB * 32;
    for (int r = blockIdx.x; r < a.requests; r += gridDim.x) {
        if (a.lens[r] > 0 && a.max_len > 0) continue;
        const int to = row_of(a, r);
        if (to < 0) continue;
        for (int i = threadIdx.x; i < row; i += kWorkThreads) store_as(a.out, a.out_dtype, (size_t)to * row + i, 0.0f);
    }
}

}  // namespace tqb
