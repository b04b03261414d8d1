// dq_kv.cu -- writing and shrinking the paged 4-bit KV cache (layout in
// dq_kv.cuh): kv_append_kernel quantizes new keys and values into their slots,
// kv_evict_kernel keeps the slots with the largest accumulated attention
// weight and moves survivors into the holes.  No counterpart in the reference
// (its scope is the linear layers); the row format and the quantizer's
// arithmetic are the reference's (src/quant_format.cuh:12-97).
#include <cfloat>
#include <climits>

#include "dq_kv.cuh"

namespace dq {

namespace {

__device__ unsigned int g_kv_error;

// ---------------------------------------------------------------------------
// Append
//
// A row of D values becomes lo = min, s = (max - lo) / 15 (1 for a row flatter
// than 1e-8), z = -lo / s and codes trunc((v - lo) / s + 1/2), with the
// operations and roundings of quantize_kernel, so a row's bytes are those of
// dq_quantize.  D/4 lanes hold one (slot pair, head): both slots' K and V rows
// are requested at once, four columns a lane, and min / max meet in shuffles.
// A pair is the granule because V words hold two neighbouring slots: with both
// slots new a lane stores whole words, else its 16-bit half.  Bound by the rows
// read and the codes written (prompts) or by one launch (a decode step).
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
    uint32_t codes;  // four codes of this lane, 4 bits each
    uint16_t s, z;
};

template <int LPR>
__device__ __forceinline__ KvRow kv_quant_row(uint2 raw) {
    const float v[4] = {h2f_bits(lo16(raw.x)), h2f_bits(hi16(raw.x)), h2f_bits(lo16(raw.y)), h2f_bits(hi16(raw.y))};
    float lo = FLT_MAX, hi = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (v[i] < lo) lo = v[i];
        if (v[i] > hi) hi = v[i];
    }
#pragma unroll
    for (int o = LPR / 2; o >= 1; o >>= 1) {
        const float l2 = __shfl_xor_sync(0xffffffffu, lo, o), h2 = __shfl_xor_sync(0xffffffffu, hi, o);
        if (l2 < lo) lo = l2;
        if (h2 > hi) hi = h2;
    }
    const float range = __fsub_rn(hi, lo);
    const float step = (range < 1e-8f) ? 1.0f : __fdiv_rn(range, 15.0f);
    const float inv = __fdiv_rn(1.0f, step);
    KvRow r;
    r.s = __half_as_ushort(__float2half_rn(step));
    r.z = __half_as_ushort(__float2half_rn(__fmul_rn(-lo, inv)));
    r.codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float t = __fadd_rn(__fmul_rn(__fsub_rn(v[i], lo), inv), 0.5f);
        // out-of-range and NaN give code 0, as quantize_kernel's conversion does
        int q = (t >= -2147483648.0f && t < 2147483648.0f) ? __float2int_rz(t) : INT_MIN;
        q = q < 0 ? 0 : (q > 15 ? 15 : q);
        r.codes |= static_cast<uint32_t>(q) << (4 * i);
    }
    return r;
}

// The four values that the cache now holds for this lane's columns.
__device__ __forceinline__ uint2 kv_values(const KvRow& r) {
    const float s = h2f_bits(r.s), z = h2f_bits(r.z);
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = __half_as_ushort(__float2half_rn(__fmul_rn(s, __fsub_rn(static_cast<float>((r.codes >> (4 * i)) & 15u), z))));
    return make_uint2(pack_h2(h[0], h[1]), pack_h2(h[2], h[3]));
}

template <int D>
__global__ void __launch_bounds__(128) kv_append_kernel(const KvAppendArgs a, const int items_per_cta) {
    constexpr int LPR = D / 4;  // lanes of one row
    const KvView& c = a.c;
    const int b = blockIdx.y;
    pdl_launch_dependents();
    pdl_wait();
    const int cap = c.max_pages * c.page_size;
    const int start = static_cast<int>(ldcg_u32((a.at ? a.at : c.lengths) + b));
    const int gone = static_cast<int>(ldcg_u32(c.evicted + b));
    int n = a.counts ? static_cast<int>(ldcg_u32(a.counts + b)) : a.tokens;
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
    const long long last = first + items_per_cta < items ? first + items_per_cta : items;
    for (long long i0 = first; i0 < last; i0 += subs) {
        const long long it = i0 + sub;
        const bool mine = it < last;
        const int pair = pair0 + static_cast<int>(mine ? it / c.heads : 0), h = static_cast<int>(mine ? it % c.heads : 0);
        bool on[2];
        uint2 kr[2], vr[2];
        int tok[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int slot = 2 * pair + e;
            tok[e] = slot - start;
            on[e] = mine && tok[e] >= 0 && tok[e] < n;
            kr[e] = vr[e] = make_uint2(0, 0);
            if (on[e]) {
                const uint16_t* kp = a.k + b * a.ks[0] + tok[e] * a.ks[1] + h * a.ks[2] + 4 * col;
                const uint16_t* vp = a.v + b * a.vs[0] + tok[e] * a.vs[1] + h * a.vs[2] + 4 * col;
                kr[e] = *reinterpret_cast<const uint2*>(kp);
                vr[e] = *reinterpret_cast<const uint2*>(vp);
            }
        }
        const int page = mine ? kv_page(c, b, 2 * pair) : 0;  // a pair never crosses a page
        KvRow kq[2], vq[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            kq[e] = kv_quant_row<LPR>(kr[e]);
            vq[e] = kv_quant_row<LPR>(vr[e]);
            if (on[e] && a.k_values) {
                const size_t o = ((static_cast<size_t>(b) * a.tokens + tok[e]) * c.heads + h) * D + 4 * col;
                *reinterpret_cast<uint2*>(a.k_values + o) = kv_values(kq[e]);
                *reinterpret_cast<uint2*>(a.v_values + o) = kv_values(vq[e]);
            }
        }
        if (!mine) continue;
        if (page < 0) { bad_page = true; continue; }
        const int off = (2 * pair) % c.page_size, row = off % kKvTokens;
        uint8_t* u = kv_unit<D>(c, page, h, off);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (!on[e]) continue;
            *reinterpret_cast<uint16_t*>(u + (row + e) * (D / 2) + 2 * col) = static_cast<uint16_t>(kq[e].codes);
            if (col == 0) {
                *reinterpret_cast<uint2*>(u + kv_param_offset(D) + 8 * (row + e)) =
                    make_uint2(pack_h2(kq[e].s, kq[e].z), pack_h2(vq[e].s, vq[e].z));
                const size_t line = kv_line(c, page, h) + off + e;
                c.mass[line] = 0.f;
                c.pos[line] = gone + 2 * pair + e;
            }
        }
        uint8_t* vw = u + kv_v_offset(D) + (row / 2) * D + 4 * col;
        if (on[0] && on[1])
            *reinterpret_cast<uint32_t*>(vw) = vq[0].codes | (vq[1].codes << 16);
        else if (on[0])
            *reinterpret_cast<uint16_t*>(vw) = static_cast<uint16_t>(vq[0].codes);
        else if (on[1])
            *reinterpret_cast<uint16_t*>(vw + 2) = static_cast<uint16_t>(vq[1].codes);
    }
    // padding tokens of the returned values are zero
    if (a.k_values) {
        const long long pad = static_cast<long long>(a.tokens - n) * c.heads * LPR;
        const size_t o = (static_cast<size_t>(b) * a.tokens + n) * c.heads * D;
        for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < pad;
             i += static_cast<long long>(gridDim.x) * blockDim.x) {
            *reinterpret_cast<uint2*>(a.k_values + o + 4 * i) = make_uint2(0, 0);
            *reinterpret_cast<uint2*>(a.v_values + o + 4 * i) = make_uint2(0, 0);
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
// One CTA per (sequence, head) with more than keep slots.  Slots are ranked by
// an order-preserving integer of their weight (protected slots first), the
// keep-th largest found by four 8-bit radix passes; ties stay in slot order.
// Survivors keep their slot unless it lies at keep or beyond: the k-th of those
// moves into the k-th hole below keep.  Sources and holes are disjoint, so the
// moves need no order among themselves, and a step that drops one slot moves
// at most one.
// ---------------------------------------------------------------------------
constexpr int kEvThreads = 1024;

struct KvEvictArgs {
    KvView c;
    int keep, recent, sink;
    int32_t* lists;  // per (sequence, head): list_cap holes, then list_cap sources
    int list_cap;
};

template <int D>
__global__ void __launch_bounds__(kEvThreads) kv_evict_kernel(const KvEvictArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t sel[2];  // chosen digit, slots above it
    __shared__ unsigned long long wsum[kEvThreads / 32 + 1];
    __shared__ int bad_any;
    const KvView& c = a.c;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait();
    bool bad = false;
    const int len = kv_length(c, b, &bad);
    const int gone = static_cast<int>(ldcg_u32(c.evicted + b));
    if (bad && tid == 0) atomicOr(&g_kv_error, kKvErrLen);
    if (tid == 0) bad_any = 0;
    __syncthreads();
    const bool work = len > a.keep;
    if (work) {
        const int newest = gone + len;
        bool bad_page = false;
        auto key = [&](int slot) -> uint32_t {
            const int page = kv_page(c, b, slot);
            if (page < 0) { bad_page = true; return 0u; }
            const size_t line = kv_line(c, page, h) + slot % c.page_size;
            const int p = static_cast<int>(ldcg_u32(c.pos + line));
            if (p >= newest - a.recent || p < a.sink) return 0xFFFFFFFFu;
            uint32_t u = __float_as_uint(__fadd_rn(ldcg_f32(c.mass + line), 0.f));  // -0 counts as 0
            u ^= (u >> 31) ? 0xFFFFFFFFu : 0x80000000u;
            return u < 0xFFFFFFFEu ? u : 0xFFFFFFFEu;
        };
        // the keep-th largest key
        uint32_t prefix = 0, mask = 0;
        int need = a.keep;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int s = tid; s < len; s += kEvThreads) {
                const uint32_t k = key(s);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (warp == 0) {
                // lane l covers digits 255 - 8l .. 248 - 8l, from the top
                uint32_t sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += hist[255 - 8 * lane - i];
                uint32_t inc = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += v;
                }
                const uint32_t before = inc - sum, want = static_cast<uint32_t>(need);
                if (before < want && want <= inc) {
                    uint32_t acc = before;
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t n = hist[255 - 8 * lane - i];
                        if (acc + n >= want) { sel[0] = 255 - 8 * lane - i; sel[1] = acc; break; }
                        acc += n;
                    }
                }
            }
            __syncthreads();
            prefix |= sel[0] << shift;
            mask |= 255u << shift;
            need -= static_cast<int>(sel[1]);
            __syncthreads();
        }
        // exclusive scan over the CTA of one 64-bit value per thread
        auto scan = [&](unsigned long long v, unsigned long long* total) {
            unsigned long long inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += t;
            }
            __syncthreads();
            if (lane == 31) wsum[warp] = inc;
            __syncthreads();
            if (warp == 0) {
                const unsigned long long w = wsum[lane];
                unsigned long long wi = w;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long t = __shfl_up_sync(0xffffffffu, wi, o);
                    if (lane >= o) wi += t;
                }
                wsum[lane] = wi - w;
                if (lane == 31) wsum[32] = wi;
            }
            __syncthreads();
            *total = wsum[32];
            return wsum[warp] + inc - v;
        };
        // slots in contiguous chunks per thread, so that ranks follow the slot order
        const int per = (len + kEvThreads - 1) / kEvThreads;
        const int s0 = min(tid * per, len), s1 = min(s0 + per, len);
        unsigned long long total = 0, eq = 0;
        for (int s = s0; s < s1; ++s) eq += key(s) == prefix;
        const unsigned long long eq0 = scan(eq, &total);
        unsigned long long cnt = 0, e = eq0;
        for (int s = s0; s < s1; ++s) {
            const uint32_t k = key(s);
            const bool stays = k > prefix || (k == prefix && e < static_cast<unsigned long long>(need));
            e += k == prefix;
            if (s < a.keep && !stays) cnt += 1ull;
            if (s >= a.keep && stays) cnt += 1ull << 32;
        }
        const unsigned long long base = scan(cnt, &total);
        const int n_moves = static_cast<int>(total & 0xFFFFFFFFull);
        int32_t* holes = a.lists + (static_cast<size_t>(b) * c.heads + h) * 2 * a.list_cap;
        int32_t* from = holes + a.list_cap;
        int hi = static_cast<int>(base & 0xFFFFFFFFull), fi = static_cast<int>(base >> 32);
        e = eq0;
        for (int s = s0; s < s1; ++s) {
            const uint32_t k = key(s);
            const bool stays = k > prefix || (k == prefix && e < static_cast<unsigned long long>(need));
            e += k == prefix;
            if (s < a.keep && !stays && hi < a.list_cap) holes[hi++] = s;
            if (s >= a.keep && stays && fi < a.list_cap) from[fi++] = s;
        }
        __syncthreads();
        // moves: D/16 lanes a slot, each 8 bytes of K and 4 half words of V
        constexpr int L = D / 16;
        for (int m = tid / L; m < n_moves; m += kEvThreads / L) {
            const int l = tid % L, to = holes[m], src = from[m];
            if (to < 0 || to >= a.keep || src < a.keep || src >= len) continue;  // lists are this call's: never taken
            const int pt = kv_page(c, b, to), ps = kv_page(c, b, src);
            if (pt < 0 || ps < 0) { bad_page = true; continue; }
            const int ot = to % c.page_size, os = src % c.page_size;
            uint8_t* ut = kv_unit<D>(c, pt, h, ot);
            const uint8_t* us = kv_unit<D>(c, ps, h, os);
            const int rt = ot % kKvTokens, rs = os % kKvTokens;
            *reinterpret_cast<uint2*>(ut + rt * (D / 2) + 8 * l) = *reinterpret_cast<const uint2*>(us + rs * (D / 2) + 8 * l);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint16_t*>(ut + kv_v_offset(D) + (rt / 2) * D + 4 * (4 * l + i) + 2 * (rt & 1)) =
                    *reinterpret_cast<const uint16_t*>(us + kv_v_offset(D) + (rs / 2) * D + 4 * (4 * l + i) + 2 * (rs & 1));
            if (l == 0) {
                *reinterpret_cast<uint2*>(ut + kv_param_offset(D) + 8 * rt) =
                    *reinterpret_cast<const uint2*>(us + kv_param_offset(D) + 8 * rs);
                const size_t lt = kv_line(c, pt, h) + ot, ls = kv_line(c, ps, h) + os;
                c.mass[lt] = c.mass[ls];
                c.pos[lt] = c.pos[ls];
            }
        }
        if (bad_page) bad_any = 1;
    }
    __syncthreads();
    if (tid == 0) {
        if (bad_any) atomicOr(&g_kv_error, kKvErrPage);
        if (atomicAdd(c.arrivals + b, 1u) == gridDim.x - 1) {
            c.arrivals[b] = 0;
            if (work) {
                c.lengths[b] = a.keep;
                c.evicted[b] = gone + len - a.keep;
            }
        }
    }
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
    const int threads = 128, subs = threads / (c.head_dim / 4);
    const long long items = (static_cast<long long>(tokens) / 2 + 1) * c.kv_heads;
    const int rounds = 4;  // items a sub-warp takes, one after another
    const int per = subs * rounds;
    const dim3 grid(static_cast<unsigned>((items + per - 1) / per), c.n_seqs);
    if (c.head_dim == 128) return launch_pdl(kv_append_kernel<128>, grid, threads, 0, stream, a, per);
    return launch_pdl(kv_append_kernel<64>, grid, threads, 0, stream, a, per);
}

size_t kv_evict_workspace(const dq_kv_cache_t& c, int keep) {
    const long long cap = static_cast<long long>(c.max_pages) * c.page_size;
    const long long n = keep < cap - keep ? keep : cap - keep;  // holes and sources of one head, at most
    if (n <= 0) return 0;
    return align256(static_cast<size_t>(c.n_seqs) * c.kv_heads * 2 * static_cast<size_t>(n) * sizeof(int32_t));
}

dq_status_t launch_kv_evict(const dq_kv_cache_t& c, int keep, int recent, int sink, void* workspace,
                            cudaStream_t stream) {
    KvEvictArgs a{};
    a.c = kv_view(c);
    a.keep = keep;
    a.recent = recent;
    a.sink = sink;
    a.lists = static_cast<int32_t*>(workspace);
    const long long cap = static_cast<long long>(c.max_pages) * c.page_size;
    a.list_cap = static_cast<int>(keep < cap - keep ? keep : cap - keep);
    const dim3 grid(c.kv_heads, c.n_seqs);
    if (c.head_dim == 128) return launch_pdl(kv_evict_kernel<128>, grid, kEvThreads, 0, stream, a);
    return launch_pdl(kv_evict_kernel<64>, grid, kEvThreads, 0, stream, a);
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
