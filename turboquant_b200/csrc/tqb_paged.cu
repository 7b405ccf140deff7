// Paged cache: block tables and slot maps from lengths, the rows that go into pages (norm, rotation and packing in one pass)
// and the rows that come back from them.  The attention over the pages is in tqb_paged_attention.cu.
#include "tqb_common.cuh"
#include "tqb_mma.cuh"
#include "tqb_paged.cuh"
#include "tqb_pqo_dequant.cuh"
#include "tqb_pqo_quant.cuh"

namespace tqb {
namespace {

// ---- block tables, slots and positions of a step ----------------------------------------------------------------------
// need_r = ceil((s_r + n_r) / P) - ceil(s_r / P); page i of them is free[F - 1 - (start_r + i)], start the exclusive sum of
// need.  Every CTA does the two prefix sums over the requests for itself (8 bytes a request from L2) and then takes its
// share of the tokens and of the new table entries; nobody waits for anybody.  What may be updated in place - lengths and
// state - is written by the CTA that finishes last, when all have read it.  Bound: launch and dependent loads: 64 requests of a
// token each 3.6 us, 211 requests, a third of which bring up to 511 tokens, 4.5 us.
constexpr int kMostCounted = 1 << 30;   // tokens of a plan or of rows that turn: an index and a grid's stride stay below 2^31
constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 256;    // tokens a CTA, up to 148 CTAs (1,024: 7.2 us for the 211 requests)

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
    int32_t* failed;   // or nullptr
    int requests, max_blocks, page_shift, capacity, free_capacity;
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
    const int status = bad ? TQB_PLAN_BAD_LENGTH : tokens > a.capacity ? TQB_PLAN_OVER_CAPACITY
                       : pages > (avail > a.free_capacity ? 0 : avail) ? TQB_PLAN_OUT_OF_PAGES : TQB_PLAN_OK;   // (no list is longer than its room)
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
        if (a.failed != nullptr) {
            const int was = status != TQB_PLAN_OK ? status : a.state[2];
            if (was != TQB_PLAN_OK) *a.failed = was;
        }
        a.state[1] = 0;
        a.state_out[0] = (int)(avail - pages);
        a.state_out[1] = 0;
        a.state_out[2] = status;
        a.state_out[3] = 0;
    }
}

// The pages of finished requests back onto the list, by one CTA: a release is rare and short.  A page that a request that stays
// holds too stays with it, and one that several ended requests hold goes back once, for the first of its entries.  Who holds what
// is told by a bit for each page of a range of 2^20, marked by the requests that stay and then by the entries in their order;
// ranges without a page to give back are passed over.  64 requests of 128 pages, one of which ends: 19 us between two events (9 for
// a kernel that gives back whatever it finds), all of which end 27 us (13); an entry a thread and round instead of four 39 us.
constexpr int kReleaseThreads = 1024;
constexpr int kMarked = 1 << 20;   // pages of a range: 128 KB of bits
constexpr int kEach = 4, kChunk = kEach * kReleaseThreads;   // entries of a thread, and of a round
constexpr int kReleaseBytes = kMarked / 8 + kChunk * 4;

struct ReleaseArgs {
    const uint8_t* mask;
    int32_t* seq;
    int32_t* table;
    long long table_stride;
    int32_t* free_pages;
    int32_t* state;
    int requests, max_blocks, free_capacity, page_shift;
};

__global__ void __launch_bounds__(kReleaseThreads) release_kernel(ReleaseArgs a) {
    extern __shared__ uint32_t s_mark[];   // [bits][the round's entries]
    int* const s_entry = reinterpret_cast<int*>(s_mark + kMarked / 32);
    __shared__ int s_start[2][TQB_PAGED_MAX_REQUESTS + 1];   // first entry of each request: of those that end, of those that stay
    __shared__ int s_high;
    __shared__ unsigned s_low;
    const int tid = threadIdx.x, R = a.requests, sh = a.page_shift;
    const long long limit = min((long long)a.max_blocks << sh, 0x7fffffffll), avail = max(a.state[0], 0);
    const int per = (R + kReleaseThreads - 1) / kReleaseThreads, r0 = min(tid * per, R), r1 = min(r0 + per, R);
    auto held = [&](int r) { return pages_of(min(max((long long)a.seq[r], 0ll), limit), sh); };
    long long going = 0, staying = 0, entries, others;
    int bad = 0;
    for (int r = r0; r < r1; ++r) {
        (a.mask[r] ? going : staying) += held(r);
        if (a.mask[r] && (a.seq[r] < 0 || a.seq[r] > limit)) bad = 1;
    }
    bad = __syncthreads_or(bad);
    block_scan2<kReleaseThreads>(going, staying, entries, others);
    int status = bad || entries > kMostCounted || others > kMostCounted ? TQB_PLAN_BAD_LENGTH : TQB_PLAN_OK;
    if (status != TQB_PLAN_OK) {
        if (tid == 0) a.state[2] = status;
        return;
    }
    for (int r = r0; r < r1; ++r) {
        s_start[0][r] = (int)going;
        s_start[1][r] = (int)staying;
        (a.mask[r] ? going : staying) += held(r);
    }
    if (tid == 0) {
        s_start[0][R] = (int)entries;
        s_start[1][R] = (int)others;
        s_low = ~0u;
        s_high = -1;
    }
    __syncthreads();
    // kEach entries from i on, of those that end (0) or stay (1); -1 behind the last one and where there is no page
    auto entries_at = [&](int side, int i, int (&page)[kEach], int32_t* (&at)[kEach]) {
        const int n = side == 0 ? (int)entries : (int)others;
        const int* start = s_start[side];
        int r = i < n ? last_not_above(start, R, i) : 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            at[k] = nullptr;
            if (i + k >= n) continue;
            while (start[r + 1] <= i + k) ++r;
            at[k] = a.table + r * a.table_stride + (i + k - start[r]);
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) page[k] = at[k] != nullptr ? max(*at[k], -1) : -1;
    };
    int page[kEach], pages = 0, high = -1;
    int32_t* at[kEach];
    unsigned low = ~0u;
    for (int i = tid * kEach; i < (int)entries; i += kChunk) {
        entries_at(0, i, page, at);
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            pages += page[k] >= 0;
            low = min(low, (unsigned)page[k]);   // (-1 is the largest)
            high = max(high, page[k]);
        }
    }
    atomicMin(&s_low, low);
    atomicMax(&s_high, high);
    auto sum = [&](int x) {
        long long v = x, none = 0, total, unused;
        __syncthreads();
        block_scan2<kReleaseThreads>(v, none, total, unused);
        return total;
    };
    const bool roomy = avail + sum(pages) <= a.free_capacity;
    const unsigned first = s_low;
    const int last = s_high;
    __syncthreads();
    // Entries whose page is not to be given back are turned over (~page), if need be after they have been counted.
    for (int pass = roomy ? 1 : 0; pass < 2; ++pass) {
        int back = 0;   // pages that are given back
        for (long long from = first; from <= last;) {
            const int words = (int)((min((long long)kMarked, last - from + 1) + 31) / 32);
            auto bit_of = [&](int x) { return x >= from && x <= last && x - from < kMarked ? (int)(x - from) : -1; };
            for (int i = tid; i < words; i += kReleaseThreads) s_mark[i] = 0;
            if (tid == 0) s_low = ~0u;
            __syncthreads();
            for (int i = tid * kEach; i < (int)others; i += kChunk) {
                entries_at(1, i, page, at);
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    const int b = bit_of(page[k]);
                    if (b >= 0) atomicOr(&s_mark[b >> 5], 1u << (b & 31));
                }
            }
            __syncthreads();
            unsigned next = ~0u;
            for (int base = 0; base < (int)entries; base += kChunk) {
                entries_at(0, base + tid * kEach, page, at);
                int b[kEach];
                unsigned taken = 0, twice = 0;   // a bit for each k
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    b[k] = bit_of(page[k]);
                    if (page[k] - from >= kMarked) next = min(next, (unsigned)page[k]);
                    if (b[k] >= 0) taken |= ((s_mark[b[k] >> 5] >> (b[k] & 31)) & 1u) << k;
                    s_entry[tid * kEach + k] = b[k];
                }
                __syncthreads();
#pragma unroll
                for (int k = 0; k < kEach; ++k)
                    if (b[k] >= 0 && !((taken >> k) & 1u)) twice |= (atomicOr(&s_mark[b[k] >> 5], 1u << (b[k] & 31)) >> (b[k] & 31)) & 1u;
                if (__syncthreads_or(twice))
#pragma unroll
                    for (int k = 0; k < kEach; ++k)   // the first of equal ones has the page
                        for (int i = 0; i < tid * kEach + k && b[k] >= 0 && !((taken >> k) & 1u); ++i) taken |= (s_entry[i] == b[k] ? 1u : 0u) << k;
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    back += b[k] >= 0 && !((taken >> k) & 1u);
                    if (((taken >> k) & 1u) && pass == 1) *at[k] = ~page[k];
                }
                __syncthreads();
            }
            atomicMin(&s_low, next);
            __syncthreads();
            from = s_low;   // (without another page: behind the last one)
            __syncthreads();
        }
        if (pass == 0 && avail + sum(back) > a.free_capacity) {
            if (tid == 0) a.state[2] = TQB_PLAN_OUT_OF_PAGES;
            return;
        }
    }
    __syncthreads();
    long long to = avail;
    for (int base = 0; base < (int)entries; base += kChunk) {
        entries_at(0, base + tid * kEach, page, at);
        long long here = 0, none = 0, total, unused;
#pragma unroll
        for (int k = 0; k < kEach; ++k) here += page[k] >= 0;
        block_scan2<kReleaseThreads>(here, none, total, unused);
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (page[k] >= 0) a.free_pages[to + here++] = page[k];
            if (at[k] != nullptr) *at[k] = -1;
        }
        to += total;
        __syncthreads();
    }
    for (int r = r0; r < r1; ++r)
        if (a.mask[r]) a.seq[r] = 0;
    if (tid == 0) {
        a.state[0] = (int)to;
        a.state[2] = TQB_PLAN_OK;
    }
}

// ---- rows into pages, with norm and rotation ---------------------------------------------------------------------------
// A warp takes a token, or half of one (a CTA a token, where there are few): its angles, its rows, its blocks.
// Angles: turns = position * inv_freq / 2 pi in f64, less whole ones, then sine and cosine in f32 (an f32 product would be off by
//   position * 2^-24, 0.06 rad at a million tokens), once for a token.
// Rows: a lane has eight elements of the first half of a row and the eight half a row behind them, so that both elements of a pair are its own; one warp
//   pass takes 32 / (D / 16) heads, and the norm's sum is shuffles away.  Passes are copied ahead to a ring in shared memory.
//   Queries leave for q_out; keys go to a tile of 32-blocks in shared memory, in their type.
// Blocks: one thread packs one 32-block of the tile, or of the values where they lie, as tqb_block_quantize does
//   (pqo_quantize_values), 16 or 12 bytes of codes.  Four lanes a block with the butterfly's last stages as shuffles needs three
//   times the instructions.
// Bound: how the rows are moved, a lane's 16-byte copies and stores and the arithmetic of their addresses: without norm and
// rotation the same kernel takes as long, with DRAM at 35 % and issue at 58 %.  8,191 tokens of 32 + 8 heads, head_dim 128, normed and
// rotated 42 us (4.0 TB/s; a plain copy of these bytes takes 32 to 36), one token 2.5 us; 6,007 tokens of 16 + 8 heads rotated and
// packed to 3 bits 28.5 us.
constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32, kRowWarpsLog = 3;
static_assert(kRowWarps == 1 << kRowWarpsLog, "");

// x / d for x below 2^31 by a multiplication: m = floor(2^(31 + s) / d) + 1 with 2^(s - 1) < d <= 2^s errs by less than 1 / d
// (Granlund and Montgomery, PLDI 1994).
struct Divisor {
    unsigned d, m, s;
    explicit Divisor(unsigned div) : d(div), m(0), s(0) {
        while ((1ull << s) < d) ++s;
        m = (unsigned)(((1ull << (31 + s)) / d) + 1);
    }
    __host__ __device__ Divisor() : d(1), m(0x80000001u), s(0) {}   // by 1
    __device__ __forceinline__ unsigned of(unsigned x) const { return (unsigned)(((unsigned long long)x * m) >> (31 + s)); }
};

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
    int at_once, token_bytes;        // rows_kernel: the CTA takes 1 << at_once tokens at a time; shared memory for a token
    int per_cta, one_more;           // tokens of a CTA; the first CTAs take one more
    unsigned total;         // append_kernel: blocks of K (or V), below 2^31 - 2^20
    Divisor by_kv;
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
    __device__ __forceinline__ void store_pieces(unsigned char* p, int k, int swizzle) const {   // elements 8 k .. of a swizzled block
        *reinterpret_cast<float4*>(p + ((2 * k) ^ swizzle) * 16) = a;
        *reinterpret_cast<float4*>(p + ((2 * k + 1) ^ swizzle) * 16) = b;
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
    __device__ __forceinline__ void store_pieces(unsigned char* p, int k, int swizzle) const { *reinterpret_cast<uint4*>(p + (k ^ swizzle) * 16) = r; }
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
    __device__ __forceinline__ void store_pieces(unsigned char* p, int k, int swizzle) const { *reinterpret_cast<uint4*>(p + (k ^ swizzle) * 16) = r; }
};

template <typename T>
struct Tile {
    static constexpr int kPitch = 32 * (int)sizeof(T) + 16;   // of a 32-block: 16-byte pieces of eight lanes in 32 banks
};
template <typename T>
__device__ __forceinline__ void load_tile(const unsigned char* p, float (&v)[32]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        Eight<T> e;
        e.load(reinterpret_cast<const T*>(p) + 8 * k);
        float x[8];
        e.get(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * k + i] = x[i];
    }
}

// Block b of a row of head h into its slot.
template <int BITS, int NB>
__device__ __forceinline__ void pack_values(const RowArgs& a, const Codebook& cb, int side, long long slot, unsigned h, unsigned b, const float (&v)[32],
                                            const float2* cells) {
    if (slot < 0 || slot >= a.num_slots) return;
    uint32_t w[4];
    const float scale = pqo_quantize_values<BITS>(v, cb, a.outer_centroid, w, cells);
    const unsigned page = (unsigned)(slot >> a.page_shift), off = (unsigned)slot & ((1u << a.page_shift) - 1);   // (rows fit in 32 bits)
    const size_t at = (size_t)(((page * (unsigned)a.kv_heads + h) << a.page_shift) + off) * NB + b;
    uint8_t* to = a.idx[side] + at * (4 * BITS);
    if (BITS == 4) {
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        uint32_t* wp = reinterpret_cast<uint32_t*>(to);
        wp[0] = w[0];
        wp[1] = w[1];
        wp[2] = w[2];
    }
    a.sc[side][at] = f32_to_f16_bits(-scale);   // outlier blocks store -scale
}

// Block b of row (token t, head h) of K or V into its slot: from the tile, or (tile == nullptr) from where the row lies.
template <typename T, int BITS, int NB>
__device__ __forceinline__ void pack_block(const RowArgs& a, const Codebook& cb, int side, long long t, unsigned h, unsigned b, const unsigned char* tile,
                                           const float2* cells) {
    const long long slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) return;
    float v[32];
    if (tile != nullptr) {
        load_tile<T>(tile, v);
    } else {
        const RowSpan& s = side == 0 ? a.k : a.v;
        load32<T>(reinterpret_cast<const T*>(s.in) + t * s.in_token + h * s.in_head + 32 * b, v);
    }
    pack_values<BITS, NB>(a, cb, side, slot, h, b, v, cells);
}

// Rows that go into their slots as they are: a block a thread, from where it lies, the next one in flight meanwhile - with two
// CTAs of an SM, that is faster than three without (16,384 tokens of 8 heads, head_dim 64: 15.3 against 17.2 us).
template <typename T, int BITS, int NB>
__global__ void __launch_bounds__(kRowThreads, 2) append_kernel(const __grid_constant__ RowArgs a, const __grid_constant__ Codebook cb) {
    __shared__ float2 s_cells[BITS == 3 ? kCells * 32 : 1];
    if (BITS == 3) {
        build_cell_table(cb, cb.n - 1, s_cells, threadIdx.x, kRowThreads);
        __syncthreads();
    }
    const unsigned total = a.total, step = gridDim.x * kRowThreads;   // of a side
    const int side = blockIdx.y;
    const RowSpan& s = side == 0 ? a.k : a.v;
    Eight<T> next[4];   // the block after this one, and its slot
    long long next_slot = -1;
    auto fetch = [&](unsigned i) {
        const unsigned row = i / NB, tok = a.by_kv.of(row);
        next_slot = a.slots[tok];
        const T* p = reinterpret_cast<const T*>(s.in) + (long long)tok * s.in_token + (row - tok * a.kv_heads) * s.in_head + 32 * (i % NB);
#pragma unroll
        for (int k = 0; k < 4; ++k) next[k].load(p + 8 * k);
    };
    unsigned i = blockIdx.x * kRowThreads + threadIdx.x;
    if (i < total) fetch(i);
    for (; i < total; i += step) {
        float v[32];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float x[8];
            next[k].get(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[8 * k + e] = x[e];
        }
        const long long slot = next_slot;
        if (total - i > step) fetch(i + step);
        const unsigned row = i / NB;
        pack_values<BITS, NB>(a, cb, side, slot, row - a.by_kv.of(row) * a.kv_heads, i % NB, v, BITS == 3 ? s_cells + (threadIdx.x & 31) : nullptr);
    }
}

// The heads of queries or keys of a token, passes `part`, part + parts, .., where only the first rot_dim elements turn; STORE:
// into the tile too.  Eight elements a lane; the partner of a pair may be in another lane.  s_cos, s_sin [rot_dim / 2].
template <typename T, int LPH, bool STORE>
__device__ __forceinline__ void do_rows_part(const RowArgs& a, const RowSpan& s, long long t, int part, int parts, const float* s_cos, const float* s_sin,
                                             unsigned char* s_tile) {
    constexpr int D = LPH * 8, HPW = 32 / LPH, NB = D / 32;
    const int lane = threadIdx.x & 31, sub = lane / LPH, l = lane % LPH;
    const bool norm = (a.flags & TQB_ROPE_NO_NORM) == 0, turn = a.rot_dim > 0, inter = (a.flags & TQB_ROPE_INTERLEAVED) != 0;
    const int hl = a.rot_dim >> 4;   // lanes of half a rotated row
    const bool turns = 8 * l < a.rot_dim;
    const int from = lane + (!turns ? 0 : l < hl ? hl : -hl);
    int h = part * HPW + sub;
    if (h - sub >= s.heads) return;
    // element e of a rotated row is v_e cos_e + v_partner sin_e, the sign of the first element's sine with it
    F2 co[4], si[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int f = inter ? 4 * l + i : 8 * (l < hl ? l : l - hl) + 2 * i;
        const int f0 = turns ? f : 0, f1 = turns && !inter ? f + 1 : f0;
        const float s0 = s_sin[f0], s1 = s_sin[f1];
        co[i] = f2(s_cos[f0], s_cos[f1]);
        si[i] = inter ? f2(-s0, s0) : l < hl ? f2(-s0, -s1) : f2(s0, s1);
    }
    F2 w[4];
    if (norm) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 1.0f;
        if (s.weight != nullptr) {
            Eight<T> e;
            e.load(reinterpret_cast<const T*>(s.weight) + 8 * l);
            e.get(x);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = f2(x[2 * i], x[2 * i + 1]);
    }
    const T* in = reinterpret_cast<const T*>(s.in) + t * s.in_token + min(h, s.heads - 1) * s.in_head + 8 * l;
    T* out = reinterpret_cast<T*>(s.out) + t * s.out_token + h * s.out_head + 8 * l;
    const int step = parts * HPW;
    const long long in_step = step * s.in_head, out_step = step * s.out_head;
    constexpr int kAhead = 1;   // passes in flight
    Eight<T> ahead[kAhead];
    auto fetch = [&](int k, int row) {   // (a lane without a head keeps to its last one)
        if (row - sub >= s.heads) return;
        ahead[k].load(in);
        if (row + step < s.heads) in += in_step;
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(k, h + k * step);
    while (h - sub < s.heads) {   // (the same for the whole warp)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (h - sub >= s.heads) break;
            Eight<T> e = ahead[k];
            fetch(k, h + kAhead * step);
            if (norm || turn) {
                float x[8];
                e.get(x);
                F2 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = f2(x[2 * i], x[2 * i + 1]);
                if (norm) {
                    F2 ss = mul2(v[0], v[0]);
#pragma unroll
                    for (int i = 1; i < 4; ++i) ss = fma2(v[i], v[i], ss);
                    const float2 u = halves(ss);
                    float sum = u.x + u.y;
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    const F2 inv = f2(rsqrtf(sum * (1.0f / D) + a.eps));   // (two steps of 2^-24)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = mul2(mul2(v[i], inv), w[i]);
                }
                if (turn) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 u = halves(v[i]);
                        F2 p;
                        if (inter) {
                            p = f2(u.y, u.x);
                        } else {
                            const float p0 = __shfl_sync(0xffffffffu, u.x, from), p1 = __shfl_sync(0xffffffffu, u.y, from);
                            p = f2(p0, p1);
                        }
                        if (turns) v[i] = fma2(v[i], co[i], mul2(p, si[i]));
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 u = halves(v[i]);
                    x[2 * i] = u.x;
                    x[2 * i + 1] = u.y;
                }
                e.set(x);
            }
            if (h < s.heads) {
                if (s.out != nullptr) e.store(out);
                if (STORE) e.store(reinterpret_cast<T*>(s_tile + (size_t)(h * NB + (l >> 2)) * Tile<T>::kPitch) + 8 * (l & 3));
            }
            out += out_step;
            h += step;
        }
    }
}

// What a warp takes in turn: `size` passes of a token, unit after unit `step` apart.
struct Units {
    int count, step, size, per_token;
    Divisor by_token;
    __device__ __forceinline__ int token_of(int unit) const { return (int)by_token.of((unsigned)unit); }
    __device__ __forceinline__ int first_pass(int unit, int token) const { return (unit - token * per_token) * size; }
};

// The same as do_rows_part where whole rows turn, or nothing does: a lane has eight elements of the first half of a row and the
// eight half a row behind them, so that both elements of a pair are its own.  Half the instructions a row (8,191 tokens of 32 + 8
// heads took 45 us with do_rows_part).
// A pass is 32 / (D / 16) heads of queries, or of keys, of a token; passes are numbered token after token, queries before keys.
// They are copied to a ring in shared memory, kDepth of them ahead; a lane reads what it has copied itself.
template <typename T, int LPH, bool STORE>
struct Rows {
    static constexpr int D = LPH * 8, LPR = LPH / 2, HPW = 32 / LPR, NB = D / 32;
    static constexpr int kDepth = 8 / (int)sizeof(T), kLane = 16 * (int)sizeof(T), kSlot = 32 * kLane;   // passes in flight, bytes a lane and a pass
    const RowArgs& a;
    const int sub, l, passes_q, passes, part, parts;   // the warp takes passes part, part + parts, .. of a unit
    const Units& u;
    int unit, pass, pass_end;                    // what is copied next
    int token;
    uint32_t to, ring;                                 // shared addresses of the lane's next slot and of its first
    const unsigned char *from, *s_ring;                // the lane's slot that is read next, and its first

    static __host__ __device__ __forceinline__ int passes_of(int heads) { return (heads + HPW - 1) / HPW; }

    __device__ __forceinline__ Rows(const RowArgs& args, const Units& units, int first, int part_, int parts_, unsigned char* space)
        : a(args), sub((threadIdx.x & 31) / LPR), l((threadIdx.x & 31) % LPR), passes_q(passes_of(args.q.heads)),
          passes(passes_q + passes_of(args.k.heads)), part(part_), parts(parts_), u(units), unit(first) {
        begin();
        s_ring = from = space + (threadIdx.x & 31) * kLane;
        to = ring = (uint32_t)__cvta_generic_to_shared(s_ring);
#pragma unroll 1
        for (int k = 0; k < kDepth; ++k) fetch();
    }
    __device__ __forceinline__ void begin() {
        token = unit < u.count ? u.token_of(unit) : 0;
        pass = u.first_pass(unit, token) + part;
        pass_end = unit < u.count ? min(passes, pass - part + u.size) : 0;
    }
    __device__ __forceinline__ void fetch() {
        if (pass < pass_end) {
            const RowSpan& s = pass < passes_q ? a.q : a.k;
            const int h = min((pass < passes_q ? pass : pass - passes_q) * HPW + sub, s.heads - 1);   // (a lane without a head reads the last one)
            const T* in = reinterpret_cast<const T*>(s.in) + token * s.in_token + h * s.in_head + 8 * l;
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
                cp_async16(to + 32 * k, reinterpret_cast<const unsigned char*>(in) + 16 * k);
                cp_async16(to + 32 * k + 16, reinterpret_cast<const unsigned char*>(in + D / 2) + 16 * k);
            }
            pass += parts;
            if (pass >= pass_end && unit < u.count) {
                unit += u.step;
                begin();
            }
        }
        cp_async_commit();
        to = to + kSlot == ring + kDepth * kSlot ? ring : to + kSlot;
    }
    // The two eights of the pass that is due; its slot is filled again.
    __device__ __forceinline__ void take(Eight<T> (&e)[2]) {
        cp_async_wait<kDepth - 1>();
        uint4 r[sizeof(T)];
#pragma unroll
        for (int k = 0; k < (int)sizeof(T); ++k) r[k] = *reinterpret_cast<const uint4*>(from + 16 * k);
        from = from + kSlot == s_ring + kDepth * kSlot ? s_ring : from + kSlot;
        __syncwarp();
        if constexpr (sizeof(T) == 2) {
            e[0].r = r[0];
            e[1].r = r[1];
        } else {
            e[0].a = *reinterpret_cast<float4*>(&r[0]);
            e[1].a = *reinterpret_cast<float4*>(&r[1]);
            e[0].b = *reinterpret_cast<float4*>(&r[2]);
            e[1].b = *reinterpret_cast<float4*>(&r[3]);
        }
        fetch();
    }
    // Passes p0, p0 + parts, .. below p1 of token t.
    __device__ __forceinline__ void run(int t, int p0, int p1, const float* s_cos, const float* s_sin, unsigned char* s_tile) {
        const bool norm = (a.flags & TQB_ROPE_NO_NORM) == 0, turn = a.rot_dim > 0, inter = (a.flags & TQB_ROPE_INTERLEAVED) != 0;
        float co[8], si[8];   // of the lane's pairs: (i, i + 8), or of neighbours
        if (turn) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int f = inter ? k * (D / 4) + 4 * l : 8 * l + 4 * k;
                const float4 c = *reinterpret_cast<const float4*>(s_cos + f), n = *reinterpret_cast<const float4*>(s_sin + f);
                co[4 * k] = c.x; co[4 * k + 1] = c.y; co[4 * k + 2] = c.z; co[4 * k + 3] = c.w;
                si[4 * k] = n.x; si[4 * k + 1] = n.y; si[4 * k + 2] = n.z; si[4 * k + 3] = n.w;
            }
        }
        Eight<T> w[2];
        bool weighted = false, fresh = true;
        for (int p = p0; p < p1; p += parts) {
            const bool keys = p >= passes_q;
            const RowSpan& s = keys ? a.k : a.q;
            const int h = (keys ? p - passes_q : p) * HPW + sub;
            if (fresh || (keys && p - parts < passes_q)) {   // a tensor begins
                fresh = false;
                weighted = norm && s.weight != nullptr;
                if (weighted) {
                    w[0].load(reinterpret_cast<const T*>(s.weight) + 8 * l);
                    w[1].load(reinterpret_cast<const T*>(s.weight) + D / 2 + 8 * l);
                }
            }
            Eight<T> e[2];
            take(e);
            if (norm || turn) {
                float x[2][8];
                e[0].get(x[0]);
                e[1].get(x[1]);
                if (norm) {
                    F2 ss = f2(0.0f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const F2 v = f2(x[i >> 2][2 * (i & 3)], x[i >> 2][2 * (i & 3) + 1]);
                        ss = fma2(v, v, ss);
                    }
                    const float2 u = halves(ss);
                    float sum = u.x + u.y;
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    const float inv = rsqrtf(sum * (1.0f / D) + a.eps);   // (two steps of 2^-24)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float wk[8];
                        if (weighted) w[k].get(wk);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[k][i] *= inv;
                            if (weighted) x[k][i] *= wk[i];
                        }
                    }
                }
                if (turn) {
                    if (inter) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float y = x[i >> 2][2 * (i & 3)], z = x[i >> 2][2 * (i & 3) + 1];
                            x[i >> 2][2 * (i & 3)] = fmaf(y, co[i], -(z * si[i]));
                            x[i >> 2][2 * (i & 3) + 1] = fmaf(z, co[i], y * si[i]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float y = x[0][i], z = x[1][i];
                            x[0][i] = fmaf(y, co[i], -(z * si[i]));
                            x[1][i] = fmaf(z, co[i], y * si[i]);
                        }
                    }
                }
                e[0].set(x[0]);
                e[1].set(x[1]);
            }
            if (h < s.heads) {
                if (s.out != nullptr) {
                    T* out = reinterpret_cast<T*>(s.out) + t * s.out_token + h * s.out_head + 8 * l;
                    e[0].store(out);
                    e[1].store(out + D / 2);
                }
                if (STORE && keys) {
                    unsigned char* at = s_tile + (size_t)(h * NB + (l >> 2)) * Tile<T>::kPitch + 8 * (l & 3) * sizeof(T);
                    e[0].store(reinterpret_cast<T*>(at));
                    e[1].store(reinterpret_cast<T*>(at + NB / 2 * Tile<T>::kPitch));
                }
            }
        }
    }
};

constexpr int kTurnWarps = 4, kTurnCtas = 5;   // of turn_kernel: CTAs of an SM
constexpr int kTurnPasses = 13;                // passes that a warp has at least, where there are more CTAs than places
constexpr int kTurnTimes = 32;                 // CTAs for each place, at most: the stride of a warp's units stays small
constexpr int kRingBytes = 4096;   // of a warp: Rows::kDepth * Rows::kSlot

// Cosines and sines of a token's angles, by `all` threads of which this is number `me`.
__device__ __forceinline__ void angles(const RowArgs& a, int t, float* s_cos, float* s_sin, int me, int all) {
    const double pos = (a.flags & TQB_ROPE_POSITIONS_64) ? (double)reinterpret_cast<const long long*>(a.positions)[t]
                                                        : (double)reinterpret_cast<const int*>(a.positions)[t];
    for (int f = me; f < a.rot_dim >> 1; f += all) {
        const double turns = pos * (double)a.inv_freq[f] * 0.15915494309189535;
        float si, co;
        sincospif((float)(2.0 * (turns - rint(turns))), &si, &co);
        s_cos[f] = co;
        s_sin[f] = si;
    }
}

// Norm and rotation alone, whole rows turning: warps take units of a token's passes in turn, neighbours neighbouring ones.
template <typename T, int LPH>
__global__ void __launch_bounds__(32 * kTurnWarps, kTurnCtas) turn_kernel(const __grid_constant__ RowArgs a, const __grid_constant__ Units u) {
    using R = Rows<T, LPH, false>;
    extern __shared__ __align__(16) unsigned char s_dyn[];   // [warp]: ring, cosines, sines
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned char* const mine = s_dyn + warp * (kRingBytes + R::D * (int)sizeof(float));
    float* const s_cos = reinterpret_cast<float*>(mine + kRingBytes);
    float* const s_sin = s_cos + R::D / 2;
    const int passes = R::passes_of(a.q.heads) + R::passes_of(a.k.heads);
    int unit = blockIdx.x * kTurnWarps + warp;
    if (unit >= u.count) return;
    R rows(a, u, unit, 0, 1, mine);
    for (; unit < u.count; unit += u.step) {
        const int t = u.token_of(unit), p = u.first_pass(unit, t);
        if (a.rot_dim > 0) {
            angles(a, t, s_cos, s_sin, lane, 32);
            __syncwarp();
        }
        rows.run(t, p, min(passes, p + u.size), s_cos, s_sin, nullptr);
        __syncwarp();   // the angles have been read
    }
}

struct NoRows {   // (do_rows_part reads for itself)
    template <typename... A>
    __device__ __forceinline__ NoRows(const A&...) {}
};

// Rows that are packed (BITS != 0), or of which only the first rot_dim elements turn (PART).  A CTA takes tokens blockIdx.x +
// i gridDim.x: eight at a time, a warp each (fewer where the tiles need more room); if not more than half of that are left, the
// warps share them, so that a last round with few tokens is a short one.  (1,183 tokens of 16 + 8 heads to 3 bits: 7.9 us; with a
// CTA for each token 14.8; 2,401 tokens 13.7 us, with a warp for each 16.5.)
template <typename T, int LPH, int BITS, bool PART>
__global__ void __launch_bounds__(kRowThreads, PART ? 3 : 2) rows_kernel(const __grid_constant__ RowArgs a, const __grid_constant__ Codebook cb) {
    constexpr int D = LPH * 8, NB = D / 32;
    using R = Rows<T, LPH, true>;
    extern __shared__ __align__(16) unsigned char s_dyn[];   // [rings][token: cosines, sines, keys' blocks]
    __shared__ float2 s_cells[BITS == 3 ? kCells * 32 : 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int half = a.rot_dim >> 1, passes = R::passes_of(a.q.heads) + R::passes_of(a.k.heads);
    if (BITS == 3) {
        build_cell_table(cb, cb.n - 1, s_cells, tid, kRowThreads);
        __syncthreads();
    }
    const int mine = a.per_cta + ((int)blockIdx.x < a.one_more ? 1 : 0);
    int shift = a.at_once, rounds = (mine >> shift) + (2 * (mine & ((1 << shift) - 1)) > 1 << shift ? 1 : 0);
#pragma unroll 1
    for (int done = 0; done < mine; rounds = 0) {
        if (rounds == 0) {
            rounds = 1;
            shift = 0;
            while (1 << shift < mine - done) ++shift;
        }
        const int parts = kRowWarps >> shift, group = warp >> (kRowWarpsLog - shift), part = warp & (parts - 1);   // `parts` warps share a token
        const int me = tid - group * parts * 32, all = parts * 32;
        auto sync = [&]() {
            if (parts == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;\n" ::"r"(1 + group), "r"(all) : "memory");
        };
        unsigned char* const space = s_dyn + (PART ? 0 : kRowWarps * kRingBytes) + (size_t)group * a.token_bytes;
        float* const s_cos = reinterpret_cast<float*>(space);
        float* const s_sin = s_cos + D / 2;
        unsigned char* const s_tile = space + (half > 0 ? D * sizeof(float) : 0);
        const int first = blockIdx.x + (done + group) * gridDim.x, step = gridDim.x << shift;
        done += rounds << shift;
        const int end = min(a.tokens, (int)(blockIdx.x + done * gridDim.x));
        const Units u{end, step, passes, 1, Divisor()};   // whole tokens
        typename std::conditional<PART, NoRows, R>::type rows(a, u, first, part, parts, s_dyn + (size_t)warp * kRingBytes);
        for (int t = first; t < end; t += step) {
            if constexpr (PART) {
                angles(a, t, s_cos, s_sin, me, all);
                sync();
                if (a.q.heads > 0) do_rows_part<T, LPH, false>(a, a.q, t, part, parts, s_cos, s_sin, s_tile);
                if (a.k.heads > 0) do_rows_part<T, LPH, BITS != 0>(a, a.k, t, part, parts, s_cos, s_sin, s_tile);
            } else {
                if (half > 0) {
                    angles(a, t, s_cos, s_sin, me, all);
                    sync();
                }
                rows.run(t, part, passes, s_cos, s_sin, s_tile);
            }
            if constexpr (BITS != 0) {
                sync();
                const int per_side = a.kv_heads * NB;
                for (int i = me; i < 2 * per_side; i += all) {   // [K, V][head][block]
                    const int side = i >= per_side ? 1 : 0, at = i - side * per_side;
                    pack_block<T, BITS, NB>(a, cb, side, t, (unsigned)at / NB, (unsigned)at % NB, side == 0 ? s_tile + (size_t)at * Tile<T>::kPitch : nullptr,
                                            BITS == 3 ? s_cells + lane : nullptr);
                }
            }
            sync();   // angles and tile are free again
        }
        if (done < mine) __syncthreads();   // other warps share a space next
    }
}

// ---- rows back from pages ----------------------------------------------------------------------------------------------
// One lane a 32-block as in tqb_block_dequantize, whose values these are; the warp's 32 blocks leave through shared memory as
// dense 512-byte stores, and the next blocks' codes are in flight.  Bound: HBM writes: 32,768 tokens of 8 heads, head_dim 128, 4
// bits to bf16 41.0 us, where a fill of the 134 MB that are written takes 35 (stages with a padded pitch, whose reads met in banks:
// 43.6; 4-bit centroids computed from the codes instead of looked up: 43.4).
struct BackArgs {
    const uint8_t* idx[2];
    const uint16_t* sc[2];
    void* out[2];
    const int64_t* slots;
    unsigned total;         // blocks of a side, below 2^31 - 2^20
    long long num_slots;
    Divisor kv_heads;
    int page_shift;
    float sign_mag;
};

template <typename T, int NB, int BITS>
__global__ void __launch_bounds__(kRowThreads, 4) back_kernel(const __grid_constant__ BackArgs a, const __grid_constant__ Codebook cb) {
    constexpr int kPitch = 32 * (int)sizeof(T), kPieces = kPitch / 16;   // 16-byte pieces of a block
    // piece k of lane l's block lies at k ^ swizzle(l): eight lanes that write the same piece, or read 128 bytes, hit all banks
    auto swizzle = [](int l) { return (sizeof(T) == 4 ? l : l >> 1) & (kPieces - 1); };
    __shared__ __align__(128) unsigned char s_tab[2 * DequantTable<BITS>::kBytes];
    __shared__ __align__(16) unsigned char s_stage[kRowThreads * kPitch];
    const int tid = threadIdx.x, lane = tid & 31, side = blockIdx.y;
    build_dequant_table<BITS>(cb, a.sign_mag, s_tab, tid, kRowThreads);
    __syncthreads();
    const uint32_t lane4 = lane * 4;
    unsigned char* stage = s_stage + (tid >> 5) * 32 * kPitch;
    const unsigned total = a.total, step = gridDim.x * kRowThreads;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    float scale = 0.0f;
    bool in = false;
    auto slot_of = [&](unsigned blk0) { return a.slots[a.kv_heads.of(min(blk0 + lane, total - 1) / NB)]; };
    auto fetch = [&](unsigned blk0, long long slot) {
        const unsigned blk = min(blk0 + lane, total - 1), row = blk / NB, tok = a.kv_heads.of(row);
        in = slot >= 0 && slot < a.num_slots;
        if (!in) return;
        const unsigned page = (unsigned)(slot >> a.page_shift), off = (unsigned)slot & ((1u << a.page_shift) - 1);   // (rows fit in 32 bits)
        const size_t at = (size_t)(((page * a.kv_heads.d + (row - tok * a.kv_heads.d)) << a.page_shift) + off) * NB + blk % NB;
        const uint8_t* p = a.idx[side] + at * (4 * BITS);
        if (BITS == 4) {
            const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        } else {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
            w[0] = __ldg(q); w[1] = __ldg(q + 1); w[2] = __ldg(q + 2);
        }
        scale = fabsf(f16_bits_to_f32(__ldg(a.sc[side] + at)));
    };
    unsigned blk0 = (blockIdx.x * kRowThreads + tid) & ~31u;
    long long slot = 0;   // of the blocks after the next
    if (blk0 < total) fetch(blk0, slot_of(blk0));
    if (blk0 + step < total) slot = slot_of(blk0 + step);
    for (; blk0 < total; blk0 += step) {
        float v[32];
        dequantize_values<BITS>(w, f2(scale), s_tab, lane4, v);
        const bool live = in;
        if (blk0 + step < total) {
            fetch(blk0 + step, slot);
            if (blk0 + 2 * step < total) slot = slot_of(blk0 + 2 * step);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = v[8 * k + i];
            Eight<T> x;
            x.set(e);
            x.store_pieces(stage + lane * kPitch, k, swizzle(lane));
        }
        if (!live) {   // a slot outside the pages
            for (int i = 0; i < kPieces; ++i) *reinterpret_cast<uint4*>(stage + lane * kPitch + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
        unsigned char* out = reinterpret_cast<unsigned char*>(a.out[side]) + (size_t)blk0 * (32 * sizeof(T)) + lane * 16;
        const bool full = blk0 + 32 <= total;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int q = 32 * i + lane;
            const uint4 r = *reinterpret_cast<const uint4*>(stage + (q / kPieces) * kPitch + ((q % kPieces) ^ swizzle(q / kPieces)) * 16);
            if (full || blk0 + q / kPieces < total) *reinterpret_cast<uint4*>(out + i * 512) = r;
        }
        __syncwarp();
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

template <typename T, int LPH, int BITS>
int launch_rows_one(RowArgs& a, const Codebook& cb, cudaStream_t s) {
    a.by_kv = Divisor((unsigned)(a.kv_heads > 0 ? a.kv_heads : 1));
    const long long blocks_of_token = (long long)a.kv_heads * (LPH / 4);
    if constexpr (BITS != 0) {
        if (a.q.heads == 0 && a.k.out == nullptr && (a.flags & TQB_ROPE_NO_NORM) != 0 && a.rot_dim == 0) {
            const long long most = ((1ll << 31) - (1 << 20)) / blocks_of_token;   // tokens of a launch
            if (most < 1) return TQB_ERR_TOO_LARGE;
            RowArgs b = a;
            for (long long done = 0; done < a.tokens; done += most) {
                const long long now = a.tokens - done < most ? a.tokens - done : most;
                b.k.in = reinterpret_cast<const T*>(a.k.in) + done * a.k.in_token;
                b.v.in = reinterpret_cast<const T*>(a.v.in) + done * a.v.in_token;
                b.slots = a.slots + done;
                b.total = (unsigned)(now * blocks_of_token);
                const long long want = (b.total + kRowThreads - 1) / kRowThreads;
                append_kernel<T, BITS, LPH / 4><<<dim3((unsigned)(want < 148 ? want : 148), 2), kRowThreads, 0, s>>>(b, cb);
                if (int e = check_launch(s)) return e;
            }
            return TQB_OK;
        }
    }
    if (a.tokens > kMostCounted) return TQB_ERR_TOO_LARGE;
    const size_t token = (BITS == 0 ? 0 : (size_t)blocks_of_token * Tile<T>::kPitch) + (a.rot_dim > 0 ? (size_t)LPH * 8 * sizeof(float) : 0);
    if (token > 128 * 1024) return TQB_ERR_UNSUPPORTED;
    a.token_bytes = (int)token;
    a.at_once = kRowWarpsLog;
    while (a.at_once > 0 && token << a.at_once > 72 * 1024) --a.at_once;
    const bool partly = a.rot_dim > 0 && a.rot_dim < LPH * 8;
    const int bytes = (int)(token << a.at_once) + (partly ? 0 : kRowWarps * kRingBytes);
    if constexpr (BITS == 0) {
        if (!partly) {
            using R = Rows<T, LPH, false>;
            const int dyn = kTurnWarps * (kRingBytes + R::D * (int)sizeof(float));
            if (int st = allow_shared<turn_kernel<T, LPH>>(dyn)) return st;
            // Half a token a unit, so that the last round is a short one (8,191 whole tokens are two or three a warp: 45 us); single
            // passes where there are few.
            const int passes = R::passes_of(a.q.heads) + R::passes_of(a.k.heads), warps = 148 * kTurnCtas * kTurnWarps;
            Units u;
            u.size = (long long)a.tokens * passes <= warps ? 1 : (passes + 1) / 2;
            u.per_token = (passes + u.size - 1) / u.size;
            const long long units = (long long)a.tokens * u.per_token;
            u.by_token = Divisor((unsigned)u.per_token);
            // A CTA for each place on the SMs, or several, as long as a warp keeps kTurnPasses passes: SMs get through their shares at
            // different speeds, and who is done early takes another CTA.  (8,191 tokens of 40 heads, head_dim 256: 76.8 us, with one
            // for each place 85.0; 16,384 of 128: 77.6 and 83.9.  But 4,096 of 128, 14 passes a warp: 22.9 us with two, 21.6 with one;
            // 6,007 with one and a half 35.6, with one 33.0.)
            const long long want = (units + kTurnWarps - 1) / kTurnWarps, times = (long long)a.tokens * passes / (warps * kTurnPasses);
            const long long most = 148 * kTurnCtas * (times > kTurnTimes ? kTurnTimes : times > 1 ? times : 1);
            const int grid = (int)(want < most ? want : most);
            u.step = grid * kTurnWarps;
            if (units + u.step >= 1ll << 31) return TQB_ERR_TOO_LARGE;   // (a unit behind the last one is the largest that is formed)
            u.count = (int)units;
            turn_kernel<T, LPH><<<grid, 32 * kTurnWarps, dyn, s>>>(a, u);
            return check_launch(s);
        }
    }
    const int most = 148 * (partly && bytes <= 64 * 1024 ? 3 : 2);
    const int grid = a.tokens < most ? a.tokens : most;
    a.per_cta = a.tokens / grid;
    a.one_more = a.tokens % grid;
    if (partly) {
        if (int st = allow_shared<rows_kernel<T, LPH, BITS, true>>(bytes, 160 * 1024)) return st;
        rows_kernel<T, LPH, BITS, true><<<grid, kRowThreads, bytes, s>>>(a, cb);
    } else if constexpr (BITS != 0) {
        if (int st = allow_shared<rows_kernel<T, LPH, BITS, false>>(bytes, 160 * 1024)) return st;
        rows_kernel<T, LPH, BITS, false><<<grid, kRowThreads, bytes, s>>>(a, cb);
    }
    return check_launch(s);
}
template <typename T, int LPH>
int launch_rows_bits(int bits, RowArgs& a, const Codebook& cb, cudaStream_t s) {
    if (bits == 0) return launch_rows_one<T, LPH, 0>(a, cb, s);
    return bits == 3 ? launch_rows_one<T, LPH, 3>(a, cb, s) : launch_rows_one<T, LPH, 4>(a, cb, s);
}
template <typename T>
int launch_rows_dim(int dim, int bits, RowArgs& a, const Codebook& cb, cudaStream_t s) {
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

int plan(const int32_t* seq_lens, const int32_t* new_tokens, int32_t num_requests, int32_t* block_table, int64_t table_stride,
         int32_t max_blocks, const int32_t* free_pages, int32_t free_capacity, int32_t* state, int32_t page_size, int64_t* slots,
         int32_t* positions, int32_t capacity, int32_t* cu, int32_t* kv_lens, int32_t* state_out, int32_t* failed, tqb_stream_t stream) {
    int st = check_plan_shape(num_requests, table_stride, max_blocks, page_size);
    if (st != TQB_OK) return st;
    if (capacity < 0 || free_capacity < 0) return TQB_ERR_INVALID_ARGUMENT;
    if (capacity > kMostCounted) return TQB_ERR_TOO_LARGE;
    if (!state || !state_out || !cu) return TQB_ERR_NULL_POINTER;
    if (num_requests > 0 && (!seq_lens || !new_tokens || !kv_lens || (max_blocks > 0 && (!block_table || !free_pages)))) return TQB_ERR_NULL_POINTER;
    if (capacity > 0 && (!slots || !positions)) return TQB_ERR_NULL_POINTER;
    PlanArgs a{seq_lens, new_tokens, block_table, table_stride, free_pages, state, slots, positions, cu, kv_lens, state_out,
               failed, num_requests, max_blocks, log2_of(page_size), capacity, free_capacity};
    int grid = (capacity + kPlanTokens - 1) / kPlanTokens;
    grid = grid < 1 ? 1 : grid > 148 ? 148 : grid;
    plan_kernel<<<grid, kPlanThreads, 0, as_stream(stream)>>>(a);
    return check_launch(as_stream(stream));
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
    return plan(seq_lens, new_tokens, num_requests, block_table, table_stride, max_blocks, free_pages, 0x7fffffff, state, page_size, slots,
                positions, capacity, cu, kv_lens, state_out, nullptr, stream);
}

int tqb_paged_plan_bounded(const int32_t* seq_lens, const int32_t* new_tokens, int32_t num_requests, int32_t* block_table,
                           int64_t table_stride, int32_t max_blocks, const int32_t* free_pages, int32_t free_capacity,
                           int32_t* state, int32_t page_size, int64_t* slots, int32_t* positions, int32_t capacity, int32_t* cu,
                           int32_t* kv_lens, int32_t* state_out, int32_t* failed, tqb_stream_t stream) {
    TQB_NVTX_RANGE();
    return plan(seq_lens, new_tokens, num_requests, block_table, table_stride, max_blocks, free_pages, free_capacity, state, page_size,
                slots, positions, capacity, cu, kv_lens, state_out, failed, stream);
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
    if ((st = allow_shared<release_kernel>(kReleaseBytes)) != TQB_OK) return st;
    const ReleaseArgs a{mask, seq_lens, block_table, table_stride, free_pages, state, num_requests, max_blocks, free_capacity, log2_of(page_size)};
    release_kernel<<<1, kReleaseThreads, kReleaseBytes, as_stream(stream)>>>(a);
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
    Codebook cb{};
    if (!block_codebook(layer->bits, TQB_MAXNORM, cb)) return TQB_ERR_UNSUPPORTED_BITS;
    const int nb = layer->head_dim / kBlock;
    const int64_t token = (int64_t)layer->num_kv_heads * nb, most = ((1ll << 31) - (1 << 20)) / token;   // blocks of a token; tokens a launch
    if (most < 1) return TQB_ERR_TOO_LARGE;
    cudaStream_t s = as_stream(stream);
    for (int64_t done = 0; done < n; done += most) {
        const int64_t now = n - done < most ? n - done : most;
        const size_t skip = (size_t)done * token * kBlock * size_of(out_dtype);
        const BackArgs a{{layer->k_indices, layer->v_indices}, {layer->k_scales, layer->v_scales},
                         {reinterpret_cast<char*>(k_out) + skip, reinterpret_cast<char*>(v_out) + skip}, slots + done, (unsigned)(now * token),
                         (long long)layer->num_pages * layer->page_size, Divisor((unsigned)layer->num_kv_heads), log2_of(layer->page_size),
                         block_sign_magnitude()};
        const long long want = (now * token + kRowThreads - 1) / kRowThreads;
        const dim3 grid((unsigned)(want < 148 * 2 ? want : 148 * 2), 2);
#define TQB_BACK(T, NB)                                                                   \
    do {                                                                                  \
        if (layer->bits == 3) back_kernel<T, NB, 3><<<grid, kRowThreads, 0, s>>>(a, cb);  \
        else back_kernel<T, NB, 4><<<grid, kRowThreads, 0, s>>>(a, cb);                   \
    } while (0)
#define TQB_BACK_DIM(T)             \
    do {                            \
        if (nb == 2) TQB_BACK(T, 2); \
        else if (nb == 4) TQB_BACK(T, 4); \
        else TQB_BACK(T, 8);        \
    } while (0)
        if (out_dtype == TQB_F32) TQB_BACK_DIM(float);
        else if (out_dtype == TQB_F16) TQB_BACK_DIM(__half);
        else TQB_BACK_DIM(__nv_bfloat16);
        if (int e = check_launch(s)) return e;
    }
#undef TQB_BACK_DIM
#undef TQB_BACK
    return TQB_OK;
}

}  // extern "C"
