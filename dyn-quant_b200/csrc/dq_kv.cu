// dq_kv.cu -- writing and shrinking the paged 4-bit KV cache (layout in
// dq_kv.cuh): kv_append_kernel quantizes new keys and values into their slots,
// kv_evict_kernel keeps the slots with the largest accumulated attention
// weight and moves survivors into the holes.  No counterpart in the reference
// (its scope is the linear layers); the row format and the quantizer's
// arithmetic are the reference's (src/quant_format.cuh:12-97).
#include <cfloat>
#include <climits>

#include <cooperative_groups.h>

#include "dq_kv.cuh"

namespace dq {

namespace {

namespace cg = cooperative_groups;

__device__ unsigned int g_kv_error;

// ---------------------------------------------------------------------------
// Append
//
// A row of D values becomes lo = min, s = (max - lo) / 15 (1 for a row flatter
// than 1e-8), z = -lo / s and codes trunc((v - lo) / s + 1/2), with the
// operations and roundings of quantize_kernel, so a finite row's bytes are
// those of dq_quantize.  D/8 lanes hold one (slot pair, head), eight columns
// each: both slots' K and V rows are requested at once in 16-byte loads.  Min
// and max of a row meet as one f16 pair (min, -max), a shuffle a step; the
// conversion to a code is one addition of 2^23 rounded down, whose low bits are
// gathered by shifted additions.  A pair is the granule because V words hold
// two neighbouring slots: with both slots new a lane stores whole words, else
// its 16-bit halves.  Bound by instructions (71% of the issue slots), then by the
// rows read and written, for prompts: 189 MB (5200 tokens of 32 heads of 128, the
// values returned) take 53 us, 3.6 TB/s; by one launch for a decode step (5 us).
// ---------------------------------------------------------------------------
struct KvAppendArgs {
    KvView c;
    const uint16_t* k;
    const uint16_t* v;
    long long ks[3], vs[3];  // strides in values: sequence, token, head
    uint16_t* k_values;      // [n_seqs][tokens][heads][D], or null
    uint16_t* v_values;
    const int32_t* counts;
    const int32_t* at;
    int tokens;
};

struct KvRow {
    uint32_t codes;  // eight codes of this lane
    uint32_t sz;     // scale | zero << 16
};

__device__ __forceinline__ uint32_t min_h2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// LPR lanes' row, eight columns each; with kValues the values that the cache now holds come back in raw.
template <int LPR, bool kValues>
__device__ __forceinline__ KvRow kv_quant_row(uint4& raw) {
    uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    const uint32_t lo2 = min_h2(min_h2(w[0], w[1]), min_h2(w[2], w[3]));
    const uint32_t hi2 = min_h2(min_h2(w[0] ^ 0x80008000u, w[1] ^ 0x80008000u), min_h2(w[2] ^ 0x80008000u, w[3] ^ 0x80008000u));
    uint32_t mm = min_h2(__byte_perm(lo2, hi2, 0x5410), __byte_perm(lo2, hi2, 0x7632));  // (min, -max)
#pragma unroll
    for (int o = LPR / 2; o >= 1; o >>= 1) mm = min_h2(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    float lo = h2f_bits(lo16(mm));
    const float range = __fsub_rn(-h2f_bits(hi16(mm)), lo);
    if (__any_sync(0xffffffffu, lo == 0.f)) {
        // zeros of both signs: the quantizer's minimum is the row's first one, whose sign the zero-point shows
        uint32_t first = 2;  // this lane's first zero: its sign, 2 where it has none
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            const uint32_t v = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
            if ((v & 0x7FFFu) == 0) first = v >> 15;
        }
        const int row = (threadIdx.x & 31) & ~(LPR - 1);  // the row's first lane
        const uint32_t has = __ballot_sync(0xffffffffu, first != 2) >> row & ((1u << LPR) - 1u);
        const uint32_t negative = __ballot_sync(0xffffffffu, first == 1) >> row;
        if (lo == 0.f) lo = (has & (0u - has) & negative) != 0 ? -0.f : 0.f;
    }
    const float step = (range < 1e-8f) ? 1.0f : __fdiv_rn(range, 15.0f);
    const float inv = __fdiv_rn(1.0f, step);
    KvRow r;
    r.sz = pack_h2(__half_as_ushort(__float2half_rn(step)), __half_as_ushort(__float2half_rn(__fmul_rn(-lo, inv))));
    const float s16 = h2f_bits(lo16(r.sz)), z16 = h2f_bits(hi16(r.sz));
    uint32_t acc = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float val[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float v = h2f_bits(e ? hi16(w[i]) : lo16(w[i]));
            // at least 0.5 (v >= lo); 15.5 at most also where the row is not finite
            const float t = fminf(__fadd_rn(__fmul_rn(__fsub_rn(v, lo), inv), 0.5f), 15.5f);
            const float c = __fadd_rz(t, 8388608.0f);  // 2^23 + trunc(t)
            acc += __float_as_uint(c) << (4 * (2 * i + e));
            if (kValues) val[e] = __fmul_rn(s16, __fsub_rn(__fsub_rn(c, 8388608.0f), z16));
        }
        if (kValues) w[i] = pack_h2(__half_as_ushort(__float2half_rn(val[0])), __half_as_ushort(__float2half_rn(val[1])));
    }
    r.codes = acc - (0x4B000000u + 0xB0000000u);  // the bits of 2^23 itself, of the terms that do not shift them out
    if (kValues) raw = make_uint4(w[0], w[1], w[2], w[3]);
    return r;
}

template <int D, bool kValues>
__global__ void __launch_bounds__(128) kv_append_kernel(const KvAppendArgs a, const int items_per_cta) {
    constexpr int LPR = D / 8;  // lanes of one row
    const KvView& c = a.c;
    const int b = blockIdx.y;
    pdl_launch_dependents();
    pdl_wait();
    const int cap = c.max_pages * c.page_size;
    const int start = ld_l2((a.at ? a.at : c.lengths) + b);
    const int gone = ld_l2(c.evicted + b);
    int n = a.counts ? ld_l2(a.counts + b) : a.tokens;
    bool bad_len = start < 0 || start > cap || n < 0 || n > a.tokens;
    const bool skip = start < 0 || start > cap;
    n = n < 0 ? 0 : (n > a.tokens ? a.tokens : n);
    if (skip) n = 0;
    else if (n > cap - start) { n = cap - start; bad_len = true; }
    if (bad_len && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(&g_kv_error, kKvErrLen);

    const int sub = threadIdx.x / LPR, subs = blockDim.x / LPR, col = threadIdx.x % LPR;
    const int pair0 = start / 2;
    const int n_pairs = n > 0 ? (start + n - 1) / 2 - pair0 + 1 : 0;
    const long long items = static_cast<long long>(n_pairs) * c.heads;
    bool bad_page = false;
    // All lanes of a warp stay in the loop together (the row reductions are shuffles of the whole warp).
    const long long first = static_cast<long long>(blockIdx.x) * items_per_cta;
    const int count = static_cast<int>(first >= items ? 0 : (items - first < items_per_cta ? items - first : items_per_cta));
    int pair = pair0 + static_cast<int>((first + sub) / c.heads), h = static_cast<int>((first + sub) % c.heads);
    for (int i0 = 0; i0 < count; i0 += subs) {
        const bool mine = i0 + sub < count;
        bool on[2];
        uint4 kr[2], vr[2];
        KvRow kq[2], vq[2];
        const int tok = 2 * pair - start;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            on[e] = mine && tok + e >= 0 && tok + e < n;
            kr[e] = vr[e] = make_uint4(0, 0, 0, 0);
            if (on[e]) {
                kr[e] = ldg_stream_v4(a.k + b * a.ks[0] + (tok + e) * a.ks[1] + h * a.ks[2] + 8 * col);
                vr[e] = ldg_stream_v4(a.v + b * a.vs[0] + (tok + e) * a.vs[1] + h * a.vs[2] + 8 * col);
            }
        }
        const int page = mine ? kv_page(c, b, 2 * pair) : 0;  // a pair never crosses a page
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            kq[e] = kv_quant_row<LPR, kValues>(kr[e]);
            vq[e] = kv_quant_row<LPR, kValues>(vr[e]);
            if (kValues && on[e]) {
                const size_t o = ((static_cast<size_t>(b) * a.tokens + tok + e) * c.heads + h) * D + 8 * col;
                *reinterpret_cast<uint4*>(a.k_values + o) = kr[e];
                *reinterpret_cast<uint4*>(a.v_values + o) = vr[e];
            }
        }
        if (mine && page < 0) bad_page = true;
        if (mine && page >= 0) {
            const int off = (2 * pair) % c.page_size, row = off % kKvTokens;
            uint8_t* u = kv_unit<D>(c, page, h, off);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (!on[e]) continue;
                *reinterpret_cast<uint32_t*>(u + (row + e) * (D / 2) + 4 * col) = kq[e].codes;
                if (col == 0) {
                    *reinterpret_cast<uint2*>(u + kv_param_offset(D) + 8 * (row + e)) = make_uint2(kq[e].sz, vq[e].sz);
                    const size_t line = kv_line(c, page, h) + off + e;
                    c.mass[line] = 0.f;
                    c.pos[line] = gone + 2 * pair + e;
                }
            }
            uint8_t* vw = u + kv_v_offset(D) + (row / 2) * D + 8 * col;  // column quads 2 col, 2 col + 1
            if (on[0] && on[1]) {
                *reinterpret_cast<uint2*>(vw) = make_uint2(__byte_perm(vq[0].codes, vq[1].codes, 0x5410),
                                                           __byte_perm(vq[0].codes, vq[1].codes, 0x7632));
            } else if (on[0] || on[1]) {
                const uint32_t x = on[0] ? vq[0].codes : vq[1].codes;
                uint16_t* half = reinterpret_cast<uint16_t*>(vw) + (on[0] ? 0 : 1);
                half[0] = lo16(x);
                half[2] = hi16(x);
            }
        }
        for (h += subs; h >= c.heads; h -= c.heads) ++pair;
    }
    // padding tokens of the returned values are zero
    if (kValues) {
        const long long pad = static_cast<long long>(a.tokens - n) * c.heads * LPR;
        const size_t o = (static_cast<size_t>(b) * a.tokens + n) * c.heads * D;
        for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < pad;
             i += static_cast<long long>(gridDim.x) * blockDim.x) {
            *reinterpret_cast<uint4*>(a.k_values + o + 8 * i) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(a.v_values + o + 8 * i) = make_uint4(0, 0, 0, 0);
        }
    }
    if (bad_page) atomicOr(&g_kv_error, kKvErrPage);
    // Every CTA of the sequence has read its length above; the last one to arrive writes the new one.
    __syncthreads();
    if (threadIdx.x == 0 && !skip) {
        if (gridDim.x == 1) {
            c.lengths[b] = start + n;
        } else if (atomicAdd(c.arrivals + b, 1u) == gridDim.x - 1) {
            c.arrivals[b] = 0;
            c.lengths[b] = start + n;
        }
    }
}

// ---------------------------------------------------------------------------
// Evict
//
// One cluster of CTAs per (sequence, head) with more than keep slots, a thread
// per unit of 16 slots: one page lookup, then its weights and positions in
// 16-byte loads.  Slots are ranked by an order-preserving integer of their
// weight (protected slots first), kept in registers.  The keep-th largest is
// found by three radix passes of 11, 11 and 10 bits over shared-memory
// histograms, summed over the cluster through distributed shared memory (beyond
// 4096 slots a CTA in several rounds, which read weights and positions again); ties
// stay in slot order (a scan of the threads' counts).  Survivors keep their slot
// unless it lies at keep or beyond: the k-th of those moves into the k-th hole
// below keep.  Sources and holes are disjoint, so the moves need no order among
// themselves, and a step that drops one slot moves at most one.  Few moves (a
// step at the cache's bound) are made by the cluster itself, many by a second
// kernel over the whole GPU; which it is goes by what a sequence's pages could hold,
// min(keep, capacity - keep).  Bound by the chain of passes (128 heads of 2049
// slots: 17 us; one CTA a head, half of its threads with a unit), then by the moves' pieces of 2 to 16 bytes (32 heads of 9000 to
// 32768 slots cut to 16384: 25 us and 31 us for 43 MB).
// ---------------------------------------------------------------------------
constexpr int kEvThreads = 256;
constexpr int kEvRadix = 2048;    // bins of a pass
constexpr int kEvBatch = 4;       // moves that a group of lanes has in flight
constexpr int kEvInline = 256;    // moves of one head, at most, that the selecting kernel makes itself
constexpr int kMvThreads = 256;

struct KvEvictArgs {
    KvView c;
    int keep, recent, sink;
    int32_t* counts;  // [n_seqs][heads] moves
    int32_t* lists;   // per (sequence, head): list_cap holes, then list_cap sources
    int list_cap;
};

// Exclusive scan of one value per thread over the CTA, and the total.
__device__ __forceinline__ uint32_t cta_scan(uint32_t v, uint32_t* wsum, uint32_t* total) {
    constexpr int W = kEvThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    __syncthreads();  // the last scan's sums have been read
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const uint32_t x = wsum[w];
        if (w < warp) before += x;
        all += x;
    }
    *total = all;
    return before + inc - v;
}

// Moves first, first + step, ... (in batches) of one (sequence, head): L lanes a slot, each 8 bytes of K codes and
// the 16 bytes of V words that hold its 16 columns.  False where a page was outside the pool.
template <int D>
__device__ __forceinline__ bool move_slots(const KvEvictArgs& a, int b, int h, int n_moves, int first, int step) {
    constexpr int L = D / 16;
    const KvView& c = a.c;
    const int32_t* holes = a.lists + (static_cast<size_t>(b) * c.heads + h) * 2 * a.list_cap;
    const int32_t* from = holes + a.list_cap;
    const int l = threadIdx.x % L, cap = c.max_pages * c.page_size;
    bool ok = true;
    for (int m0 = first; m0 < n_moves; m0 += step) {
        uint2 kc[kEvBatch], par[kEvBatch];
        uint4 vc[kEvBatch];
        float w[kEvBatch];
        int p[kEvBatch], to[kEvBatch], pt[kEvBatch], src[kEvBatch], ps[kEvBatch];
        bool on[kEvBatch];
#pragma unroll
        for (int j = 0; j < kEvBatch; ++j) {
            on[j] = m0 + j < n_moves;
            to[j] = on[j] ? ld_l2(holes + m0 + j) : 0;
            src[j] = on[j] ? ld_l2(from + m0 + j) : a.keep;
        }
#pragma unroll
        for (int j = 0; j < kEvBatch; ++j) {
            on[j] = on[j] && to[j] >= 0 && to[j] < a.keep && src[j] >= a.keep && src[j] < cap;  // (lists of this call: always)
            ps[j] = on[j] ? kv_page(c, b, src[j]) : 0;
            pt[j] = on[j] ? kv_page(c, b, to[j]) : 0;
        }
#pragma unroll
        for (int j = 0; j < kEvBatch; ++j) {
            if (ps[j] < 0 || pt[j] < 0) { ok = false; on[j] = false; }
            if (on[j]) {
                const int os = src[j] % c.page_size, rs = os % kKvTokens;
                const uint8_t* us = kv_unit<D>(c, ps[j], h, os);
                kc[j] = *reinterpret_cast<const uint2*>(us + rs * (D / 2) + 8 * l);
                vc[j] = *reinterpret_cast<const uint4*>(us + kv_v_offset(D) + (rs / 2) * D + 16 * l);
                if (rs & 1) vc[j] = make_uint4(vc[j].x >> 16, vc[j].y >> 16, vc[j].z >> 16, vc[j].w >> 16);
                if (l == 0) {
                    par[j] = *reinterpret_cast<const uint2*>(us + kv_param_offset(D) + 8 * rs);
                    const size_t ls = kv_line(c, ps[j], h) + os;
                    w[j] = ld_l2(c.mass + ls);
                    p[j] = ld_l2(c.pos + ls);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kEvBatch; ++j) {
            if (!on[j]) continue;
            const int ot = to[j] % c.page_size, rt = ot % kKvTokens;
            uint8_t* ut = kv_unit<D>(c, pt[j], h, ot);
            *reinterpret_cast<uint2*>(ut + rt * (D / 2) + 8 * l) = kc[j];
            uint16_t* vt = reinterpret_cast<uint16_t*>(ut + kv_v_offset(D) + (rt / 2) * D + 16 * l) + (rt & 1);
            vt[0] = static_cast<uint16_t>(vc[j].x);
            vt[2] = static_cast<uint16_t>(vc[j].y);
            vt[4] = static_cast<uint16_t>(vc[j].z);
            vt[6] = static_cast<uint16_t>(vc[j].w);
            if (l == 0) {
                *reinterpret_cast<uint2*>(ut + kv_param_offset(D) + 8 * rt) = par[j];
                const size_t lt = kv_line(c, pt[j], h) + ot;
                c.mass[lt] = w[j];
                c.pos[lt] = p[j];
            }
        }
    }
    return ok;
}

template <int D>
__global__ void __launch_bounds__(kEvThreads) kv_evict_kernel(const KvEvictArgs a) {
    __shared__ __align__(16) uint32_t local[2][kEvRadix];  // this CTA's counts: of the first two passes, of the last
    __shared__ __align__(16) uint32_t hists[3][kEvRadix];  // the cluster's counts, one a pass
    __shared__ uint32_t sel[2];   // chosen digit, slots above it
    __shared__ __align__(8) uint32_t sums[2];  // of this CTA: holes, sources
    __shared__ uint32_t got[3];    // what the cluster's other CTAs say
    __shared__ uint32_t wsum[kEvThreads / 32];
    const KvView& c = a.c;
    const cg::cluster_group cluster = cg::this_cluster();
    const int cs = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int h = blockIdx.x / cs, b = blockIdx.y, tid = threadIdx.x;
    auto meet = [&]() {
        if (cs > 1) cluster.sync();
        else __syncthreads();
    };
    pdl_launch_dependents();
    pdl_wait();
    bool bad = false, page_ok = true;
    const int len = kv_length(c, b, &bad);
    const int gone = ld_l2(c.evicted + b);
    if (bad && tid == 0) atomicOr(&g_kv_error, kKvErrLen);
    bool work = len > a.keep;
    int n_moves = 0;
    const int newest = gone + len;
    const int units = (len + kKvTokens - 1) / kKvTokens, share = (units + cs - 1) / cs, rounds = (share + kEvThreads - 1) / kEvThreads;
    uint32_t k[kKvTokens];
    int n = 0, slot0 = 0;  // this thread's unit of the round: its slots in use, the first of them
    auto fetch = [&](int round) {
        const int i = round * kEvThreads + tid;
        slot0 = (rank * share + i) * kKvTokens;
        n = i >= share || len - slot0 < 0 ? 0 : (len - slot0 > kKvTokens ? kKvTokens : len - slot0);
        const int page = n > 0 ? kv_page(c, b, slot0) : -1;
#pragma unroll
        for (int j = 0; j < kKvTokens; ++j) k[j] = 0u;
        if (page >= 0) {
            const size_t line = kv_line(c, page, h) + slot0 % c.page_size;
            uint32_t w[kKvTokens], p[kKvTokens];
            const bool wide = ((reinterpret_cast<uintptr_t>(c.mass) | reinterpret_cast<uintptr_t>(c.pos)) & 15u) == 0;
#pragma unroll
            for (int j = 0; j < kKvTokens; j += 4) {
                if (wide) {
                    const uint4 x = ld_l2_v4(c.mass + line + j), y = ld_l2_v4(c.pos + line + j);
                    w[j] = x.x; w[j + 1] = x.y; w[j + 2] = x.z; w[j + 3] = x.w;
                    p[j] = y.x; p[j + 1] = y.y; p[j + 2] = y.z; p[j + 3] = y.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[j + e] = __float_as_uint(ld_l2(c.mass + line + j + e));
                        p[j + e] = static_cast<uint32_t>(ld_l2(c.pos + line + j + e));
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kKvTokens; ++j) {
                uint32_t u = __float_as_uint(__fadd_rn(__uint_as_float(w[j]), 0.f));  // -0 counts as 0
                u ^= (u >> 31) ? 0xFFFFFFFFu : 0x80000000u;
                const int at = static_cast<int>(p[j]);
                k[j] = (at >= newest - a.recent || at < a.sink) ? 0xFFFFFFFFu : (u < 0xFFFFFFFEu ? u : 0xFFFFFFFEu);
            }
        }
    };
    if (work) {
        for (int i = 4 * tid; i < 2 * kEvRadix; i += 4 * kEvThreads) *reinterpret_cast<uint4*>(&local[0][0] + i) = make_uint4(0, 0, 0, 0);
        for (int i = 4 * tid; i < 3 * kEvRadix; i += 4 * kEvThreads) *reinterpret_cast<uint4*>(&hists[0][0] + i) = make_uint4(0, 0, 0, 0);
        // A sequence with a page outside the pool is left as it is: a slot that is not there can neither be ranked nor
        // take a survivor.  Every CTA looks at all of its pages, so that they agree.
        bool there = true;
        for (int i = tid; i * c.page_size < len; i += kEvThreads) there &= kv_page(c, b, i * c.page_size) >= 0;
        if (rounds == 1) fetch(0);
        if (cs > 1) cluster.sync();
        work = page_ok = __syncthreads_and(there);
    }
    if (work) {
        // the keep-th largest key
        uint32_t prefix = 0, mask = 0;
        int need = a.keep;
        constexpr int B = kEvRadix / kEvThreads;  // bins of a thread
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
            const uint32_t bins = pass == 2 ? 1023u : 2047u;
            uint32_t* mine = local[pass == 2 ? 1 : 0];
            for (int r = 0; r < rounds; ++r) {
                if (rounds > 1) fetch(r);
#pragma unroll
                for (int i = 0; i < kKvTokens; ++i)
                    if (i < n && (k[i] & mask) == prefix) atomicAdd(&mine[(k[i] >> shift) & bins], 1u);
            }
            __syncthreads();
            // bins top .. top + B - 1, threads counted from the largest bin; the few that are not empty go to
            // every CTA of the cluster
            const int top = kEvRadix - B - B * tid;
            uint32_t cnt[B], sum = 0;
#pragma unroll
            for (int i = 0; i < B; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(mine + top + i);
                cnt[i] = v.x; cnt[i + 1] = v.y; cnt[i + 2] = v.z; cnt[i + 3] = v.w;
                if (pass == 0) *reinterpret_cast<uint4*>(mine + top + i) = make_uint4(0, 0, 0, 0);
            }
            if (cs > 1) {
#pragma unroll
                for (int i = 0; i < B; ++i)
                    if (cnt[i] != 0)
                        for (int r = 0; r < cs; ++r) atomicAdd(cluster.map_shared_rank(&hists[pass][top + i], r), cnt[i]);
                meet();
#pragma unroll
                for (int i = 0; i < B; i += 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(&hists[pass][top + i]);
                    cnt[i] = v.x; cnt[i + 1] = v.y; cnt[i + 2] = v.z; cnt[i + 3] = v.w;
                }
            }
#pragma unroll
            for (int i = 0; i < B; ++i) sum += cnt[i];
            uint32_t total;
            const uint32_t before = cta_scan(sum, wsum, &total), want = static_cast<uint32_t>(need);
            if (before < want && want <= before + sum) {
                uint32_t acc = before;
                bool open = true;
#pragma unroll
                for (int i = B - 1; i >= 0; --i) {
                    if (open && acc + cnt[i] >= want) { sel[0] = top + i; sel[1] = acc; open = false; }
                    acc += cnt[i];
                }
            }
            __syncthreads();
            prefix |= sel[0] << shift;
            mask |= bins << shift;
            need -= static_cast<int>(sel[1]);
        }
        // slots equal to the threshold: how many before this thread's (in the round, then before the CTA)
        uint32_t total, eq_at = 0;
        auto equal = [&]() {
            uint32_t e = 0;
#pragma unroll
            for (int i = 0; i < kKvTokens; ++i) e += i < n && k[i] == prefix;
            return e;
        };
        if (rounds == 1) eq_at = cta_scan(equal(), wsum, &total);
        uint32_t eq0 = 0;
        if (cs > 1) {  // the last pass counted them: the threshold's bin in the CTAs before
            if (tid < 32) {
                const uint32_t x = tid < rank ? cluster.map_shared_rank(&local[1][0], tid)[prefix & 1023u] : 0u;
                const uint32_t all = __reduce_add_sync(0xffffffffu, x);
                if (tid == 0) got[0] = all;
            }
            __syncthreads();
            eq0 = got[0];
        }
        // bit i of stay: slot i of the unit stays; holes | sources << 16 of the unit
        uint32_t stay = 0;
        auto decide = [&](uint32_t e) -> uint32_t {
            stay = 0;
#pragma unroll
            for (int i = 0; i < kKvTokens; ++i) {
                const bool same = k[i] == prefix;
                if (i < n && (k[i] > prefix || (same && e < static_cast<uint32_t>(need)))) stay |= 1u << i;
                e += same && i < n;
            }
            const int low = a.keep - slot0 < 0 ? 0 : (a.keep - slot0 > kKvTokens ? kKvTokens : a.keep - slot0);
            const uint32_t below = (1u << low) - 1u, used = (1u << n) - 1u;
            return __popc(~stay & below & used) | (__popc(stay & ~below) << 16);
        };
        uint32_t holes_n = 0, from_n = 0, at = 0, eq_run = eq0;
        for (int r = 0; r < rounds; ++r) {
            if (rounds > 1) {
                fetch(r);
                eq_at = cta_scan(equal(), wsum, &total);
            }
            const uint32_t mine = decide(eq_run + eq_at);
            if (rounds > 1) eq_run += total;
            at = cta_scan(mine, wsum, &total);  // at most 16 x 256 of either: no carry between the halves
            holes_n += total & 0xFFFFu;
            from_n += total >> 16;
        }
        uint32_t holes_at = 0, from_at = 0;
        n_moves = static_cast<int>(holes_n);
        if (cs > 1) {
            if (tid == 0) { sums[0] = holes_n; sums[1] = from_n; }
            meet();
            if (tid < 32) {
                uint2 x = make_uint2(0u, 0u);
                if (tid < cs) x = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&sums[0], tid));
                const uint32_t all = __reduce_add_sync(0xffffffffu, x.x);
                const uint32_t h0 = __reduce_add_sync(0xffffffffu, tid < rank ? x.x : 0u);
                const uint32_t f0 = __reduce_add_sync(0xffffffffu, tid < rank ? x.y : 0u);
                if (tid == 0) { got[0] = all; got[1] = h0; got[2] = f0; }
            }
            __syncthreads();
            n_moves = static_cast<int>(got[0]);
            holes_at = got[1];
            from_at = got[2];
        }
        int32_t* holes = a.lists + (static_cast<size_t>(b) * c.heads + h) * 2 * a.list_cap;
        int32_t* from = holes + a.list_cap;
        eq_run = eq0;
        for (int r = 0; r < rounds; ++r) {
            if (rounds > 1) {
                fetch(r);
                eq_at = cta_scan(equal(), wsum, &total);
                const uint32_t mine = decide(eq_run + eq_at);
                eq_run += total;
                at = cta_scan(mine, wsum, &total);
            }
            uint32_t x = holes_at + (at & 0xFFFFu), y = from_at + (at >> 16);
            const int low = a.keep - slot0 < 0 ? 0 : (a.keep - slot0 > kKvTokens ? kKvTokens : a.keep - slot0);
            const uint32_t below = (1u << low) - 1u, used = (1u << n) - 1u;
            for (uint32_t m = ~stay & below & used; m; m &= m - 1, ++x)
                if (x < static_cast<uint32_t>(a.list_cap)) holes[x] = slot0 + __ffs(m) - 1;
            for (uint32_t m = stay & ~below; m; m &= m - 1, ++y)
                if (y < static_cast<uint32_t>(a.list_cap)) from[y] = slot0 + __ffs(m) - 1;
            holes_at += total & 0xFFFFu;
            from_at += total >> 16;
        }
        meet();
        if (a.list_cap <= kEvInline) {
            constexpr int L = D / 16;
            if (!move_slots<D>(a, b, h, n_moves, (rank * kEvThreads + tid) / L * kEvBatch, cs * kEvThreads / L * kEvBatch))
                page_ok = false;
        }
    }
    if (!page_ok) atomicOr(&g_kv_error, kKvErrPage);
    __syncthreads();
    if (tid == 0) {
        if (rank == 0 && a.list_cap > kEvInline) a.counts[b * c.heads + h] = n_moves;
        // every CTA of the sequence has read its length: the last one to arrive writes the new one
        if (atomicAdd(c.arrivals + b, 1u) == gridDim.x - 1) {
            c.arrivals[b] = 0;
            if (work) {
                c.lengths[b] = a.keep;
                c.evicted[b] = gone + len - a.keep;
            }
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kMvThreads, 4) kv_move_kernel(const KvEvictArgs a) {
    constexpr int L = D / 16;
    pdl_launch_dependents();
    pdl_wait();
    const int h = blockIdx.y, b = blockIdx.z, n = ld_l2(a.counts + b * a.c.heads + h);
    const int first = (static_cast<int>(blockIdx.x * kMvThreads + threadIdx.x)) / L * kEvBatch;
    if (first < n && !move_slots<D>(a, b, h, n, first, static_cast<int>(gridDim.x) * kMvThreads / L * kEvBatch))
        atomicOr(&g_kv_error, kKvErrPage);
}

// CTAs per (sequence, head): as many as fill the GPU (four on an SM), at most 8 and no more than give every CTA
// 2048 slots of a full sequence.
int evict_cluster(const dq_kv_cache_t& c, int sm_count) {
    const long long pairs = static_cast<long long>(c.n_seqs) * c.kv_heads, cap = static_cast<long long>(c.max_pages) * c.page_size;
    int cs = 1;
    while (cs < 8 && pairs * cs * 2 <= 4ll * sm_count && cap >= 2048ll * cs * 2) cs *= 2;
    return cs;
}

template <int D>
dq_status_t evict(const dq_kv_cache_t& c, const KvEvictArgs& a, int sm_count, cudaStream_t stream) {
    const int cs = evict_cluster(c, sm_count);
    const dq_status_t st = launch_pdl(kv_evict_kernel<D>, dim3(c.kv_heads * cs, c.n_seqs), kEvThreads, 0, stream, cs, a);
    if (st != DQ_OK || a.list_cap <= kEvInline) return st;
    // a batch per group of lanes: heads differ in their moves, and most CTAs of the grid find none
    constexpr int kPer = kMvThreads / (D / 16) * kEvBatch;
    return launch_pdl(kv_move_kernel<D>, dim3((a.list_cap + kPer - 1) / kPer, c.kv_heads, c.n_seqs), kMvThreads, 0, stream, 1, a);
}

}  // namespace

dq_status_t launch_kv_append(const dq_kv_cache_t& c, const uint16_t* k, const int64_t ks[3], const uint16_t* v,
                             const int64_t vs[3], int tokens, const int32_t* counts, const int32_t* at,
                             uint16_t* k_values, uint16_t* v_values, cudaStream_t stream) {
    KvAppendArgs a{};
    a.c = kv_view(c);
    a.k = k;
    a.v = v;
    for (int i = 0; i < 3; ++i) { a.ks[i] = ks[i]; a.vs[i] = vs[i]; }
    a.k_values = k_values;
    a.v_values = v_values;
    a.counts = counts;
    a.at = at;
    a.tokens = tokens;
    const int threads = 128, subs = threads / (c.head_dim / 8);
    const long long items = (static_cast<long long>(tokens) / 2 + 1) * c.kv_heads;
    const int per = subs * 4;  // a sub-warp takes four items, one after another
    const dim3 grid(static_cast<unsigned>((items + per - 1) / per), c.n_seqs);
    const bool values = k_values != nullptr;
    if (c.head_dim == 128)
        return values ? launch_pdl(kv_append_kernel<128, true>, grid, threads, 0, stream, 1, a, per)
                      : launch_pdl(kv_append_kernel<128, false>, grid, threads, 0, stream, 1, a, per);
    return values ? launch_pdl(kv_append_kernel<64, true>, grid, threads, 0, stream, 1, a, per)
                  : launch_pdl(kv_append_kernel<64, false>, grid, threads, 0, stream, 1, a, per);
}

// Holes and sources of one head, at most.
static long long evict_list_cap(const dq_kv_cache_t& c, int keep) {
    const long long cap = static_cast<long long>(c.max_pages) * c.page_size, n = keep < cap - keep ? keep : cap - keep;
    return n < 0 ? 0 : n;
}

static size_t evict_lists_bytes(const dq_kv_cache_t& c, int keep) {
    return align256(static_cast<size_t>(c.n_seqs) * c.kv_heads * 2 * static_cast<size_t>(evict_list_cap(c, keep)) * sizeof(int32_t));
}

size_t kv_evict_workspace(const dq_kv_cache_t& c, int keep) {
    const size_t lists = evict_lists_bytes(c, keep);
    return lists == 0 ? 0 : lists + align256(static_cast<size_t>(c.n_seqs) * c.kv_heads * sizeof(int32_t));
}

dq_status_t launch_kv_evict(const dq_kv_cache_t& c, int keep, int recent, int sink, void* workspace,
                            cudaStream_t stream) {
    DeviceInfo di;
    const dq_status_t st = device_info(&di);
    if (st != DQ_OK) return st;
    KvEvictArgs a{};
    a.c = kv_view(c);
    a.keep = keep;
    a.recent = recent;
    a.sink = sink;
    a.lists = static_cast<int32_t*>(workspace);
    a.counts = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + evict_lists_bytes(c, keep));
    a.list_cap = static_cast<int>(evict_list_cap(c, keep));
    return c.head_dim == 128 ? evict<128>(c, a, di.sm_count, stream) : evict<64>(c, a, di.sm_count, stream);
}

dq_status_t read_kv_error(uint32_t* word, bool clear) {
    unsigned int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_kv_error, sizeof(v));
    if (e == cudaSuccess && clear && v) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_kv_error, &zero, sizeof(zero));
    }
    if (e != cudaSuccess) { set_cuda_error(e); return DQ_ERR_CUDA; }
    *word = v;
    return DQ_OK;
}

}  // namespace dq
