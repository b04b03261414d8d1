// dq_kv_attend.cu -- attention of the newest tokens over the paged 4-bit KV
// cache (layout in dq_kv.cuh).  No counterpart in the reference.
//
//   out_r = sum_j p_rj V_j,  p_rj = softmax_j(scale <q_r, K_j>),  K_j = s_j (c_j - z_j), V_j alike
//
// One pass over the cache with the running maximum and sum of the softmax.
// Rows r = (query token, query head of the KV head) share the KV head's units.
//
// Work split: the units of all (sequence, KV head, row tile) jobs form one
// list, cut into equal runs, one per warp of a persistent grid, so ragged
// lengths, few sequences and long ones all fill the GPU.  Each warp streams
// its run through a ring of bulk copies of its own; job borders do not
// interrupt the stream.  A job inside one run is finished there; the others
// leave their partial sums (maximum, sum, unnormalised output) in the
// workspace, which kv_combine_kernel joins in warp order.
//
// Products (mma.sync.m16n8k16, f16 x f16 -> f32) are transposed, so that the 16
// slots of a unit are the MMA's rows and the query rows its 8 columns:
//   S^T = K Q^T   A = 16 slots x 16 columns of K, B = Q^T
//   O^T = V^T P^T A = 16 columns of V x 16 slots, B = P^T
// A decode step has at most 8 rows per KV head, so nothing of an MMA is idle,
// and a lane's S values (slots g, g + 8; rows 2t, 2t + 1) lie in the lanes that
// hold its O columns' rows: maxima, sums and rescaling stay in the lane.
// Codes become f16 integers c - 8 exactly: (bits 4..7 | 0x5400) is 64 + c, one
// f16x2 subtraction takes 72.  Scales and zeros are applied in FP32:
//   S   = s_k (D - (z_k - 8) sum q),  D the MMA's sum of q (c - 8)
//   O   = sum p' (c - 8) - sum p' (z_v - 8),  p' = p s_v w
// p' is the only rounding to FP16 besides the output's: p <= 2^8 (the maximum
// is taken again only when a score passes it by 8) and w is the power of two
// that brings the largest s_v seen to at most 2^7, so p' <= 2^15 and small
// weights keep their 11 bits down to 2^-29 of the largest.
#include "dq_kv.cuh"

namespace dq {

namespace {

__device__ unsigned int g_kv_attend_error;

constexpr int kAtWarps = 4;           // warps per CTA
constexpr int kAtMaxWarps = 2560;     // bound on the grid's warps (workspace sizing)
constexpr float kNone = -1e30f;       // running maximum of a row that has seen no key
constexpr float kLazy = 8.0f;         // a score passes the running maximum by this much (log2) before it moves

struct KvAttendArgs {
    KvView c;
    const uint16_t* q;
    uint16_t* out;
    long long qs[3], os[3];  // strides in values: sequence, token, head
    float* lse;              // [n_seqs][tokens][q_heads] natural log, or null
    float* lse2;             // workspace: the same in log2 (mass pass), or null
    const int32_t* counts;
    float* part;             // [warps][2][rows][D]
    float* part_ml;          // [warps][2][rows][2]
    int tokens, group, n_rt; // query tokens, query heads per KV head, row tiles
    float scale2;            // scale * log2(e)
    int depth;               // ring slots per warp
};

// The list of units: pre[b] = units of the sequences before b, a job being
// ulen[b] units of one (sequence, KV head, row tile).
struct Plan {
    const long long* pre;
    const int* len;
    long long total;
    long long base;  // units per warp; the first rem warps take one more
    int rem;
    int jobs;        // per sequence
};

// Bytes of the plan in shared memory.
__host__ __device__ inline int plan_bytes(int n_seqs) { return ((n_seqs + 1) * 8 + n_seqs * 4 + 127) / 128 * 128; }

__device__ __forceinline__ long long warp_start(const Plan& p, long long w) {
    return w * p.base + (w < p.rem ? w : p.rem);
}
__device__ __forceinline__ long long warp_of(const Plan& p, long long u) {
    const long long cut = p.rem * (p.base + 1);
    return u < cut ? u / (p.base + 1) : p.rem + (u - cut) / p.base;
}

// Built by every CTA from the lengths (a few KB from L2); all threads call it.
template <int NT>
__device__ Plan make_plan(const KvView& c, int jobs, int warps, char* smem, unsigned int* err) {
    long long* pre = reinterpret_cast<long long*>(smem);
    int* lens = reinterpret_cast<int*>(smem + (c.n_seqs + 1) * 8);
    __shared__ long long wtot[NT / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long run = 0;
    for (int b0 = 0; b0 < c.n_seqs; b0 += NT) {
        const int b = b0 + tid;
        long long v = 0;
        if (b < c.n_seqs) {
            bool bad = false;
            const int n = kv_length(c, b, &bad);
            if (bad && err) atomicOr(err, kKvErrLen);
            lens[b] = n;
            v = static_cast<long long>((n + kKvTokens - 1) / kKvTokens) * jobs;
        }
        long long inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        if (lane == 31) wtot[warp] = inc;
        __syncthreads();
        long long before = run;
        for (int w = 0; w < NT / 32; ++w) {
            if (w < warp) before += wtot[w];
            run += wtot[w];
        }
        if (b < c.n_seqs) pre[b] = before + inc - v;
        __syncthreads();
    }
    if (tid == 0) pre[c.n_seqs] = run;
    __syncthreads();
    Plan p;
    p.pre = pre;
    p.len = lens;
    p.total = run;
    p.base = run / warps;
    p.rem = static_cast<int>(run - p.base * warps);
    p.jobs = jobs;
    return p;
}

// The sequence of unit u (u < total): the last b with pre[b] <= u that has units.
__device__ __forceinline__ int seq_of(const Plan& p, int n_seqs, long long u) {
    int lo = 0, hi = n_seqs;  // pre[lo] <= u < pre[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.pre[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

// f16 pairs (c - 8) of the nibbles at bits 4..7 and 20..23.
__device__ __forceinline__ uint32_t centred(uint32_t w) {
    return hsub2_u32(lop3_and_or(w, 0x00F000F0u, 0x54005400u), 0x54805480u);  // (64 + c) - 72
}

// An 8x8 matrix of b16 in the MMA layout, transposed across the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ uint32_t pack_f32(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float lane_max_g(float v) {  // over the lanes g of one t
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float lane_sum_g(float v) {
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// B fragments of 8 NT query rows and what the scores need of them.
template <int D, int NT>
struct QueryTile {
    uint32_t f[NT][D / 8];  // per 8-column word: (0,4), (1,5), (2,6), (3,7)
    float sum[NT][2];       // sum of q over the columns, rows 2t and 2t + 1
    int lim[NT][2];         // keys that rows 2t and 2t + 1 see
    int min_lim, max_lim;   // over the tile's rows

    // row r of the job: query token r / group, head h * group + r % group
    __device__ __forceinline__ void load(const KvAttendArgs& a, int b, int h, int rt, int len) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const int rows = a.tokens * a.group;
        const int cnt = a.counts ? min(max(static_cast<int>(ldcg_u32(a.counts + b)), 0), a.tokens) : a.tokens;
        int lo = len, hi = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = (rt * NT + nt) * 8 + g;
            const int tok = r / a.group;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (r < rows && tok < cnt)
                    w = ldcg_v4(a.q + b * a.qs[0] + tok * a.qs[1] + (h * a.group + r % a.group) * a.qs[2] + (D / 4) * t + 8 * i);
                f[nt][4 * i] = __byte_perm(w.x, w.z, 0x5410);
                f[nt][4 * i + 1] = __byte_perm(w.x, w.z, 0x7632);
                f[nt][4 * i + 2] = __byte_perm(w.y, w.w, 0x5410);
                f[nt][4 * i + 3] = __byte_perm(w.y, w.w, 0x7632);
                const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) s += h2f_bits(lo16(v[k])) + h2f_bits(hi16(v[k]));
            }
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            // keys of row r: the query tokens are the sequence's last cnt; padding rows see all keys (unused)
            int l = len;
            if (r < rows) {
                l = tok < cnt ? min(max(len - cnt + tok + 1, 0), len) : 0;
                lo = min(lo, l);
                hi = max(hi, l);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sum[nt][e] = __shfl_sync(0xffffffffu, s, 8 * t + 4 * e);
                lim[nt][e] = __shfl_sync(0xffffffffu, l, 8 * t + 4 * e);
            }
        }
        min_lim = __reduce_min_sync(0xffffffffu, lo);
        max_lim = __reduce_max_sync(0xffffffffu, hi);
    }
};

// D of one unit: the MMA's sum of q (c - 8) for slots g, g + 8 and rows 2t, 2t + 1.
template <int D, int NT>
__device__ __forceinline__ void score_mma(uint32_t unit, const QueryTile<D, NT>& q, float (&s)[NT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t k0[D / 32], k1[D / 32];
    if (D == 128) {
        const uint4 x = lds_v4(unit + g * 64 + t * 16), y = lds_v4(unit + (g + 8) * 64 + t * 16);
        k0[0] = x.x; k0[1] = x.y; k0[D / 32 - 2] = x.z; k0[D / 32 - 1] = x.w;
        k1[0] = y.x; k1[1] = y.y; k1[D / 32 - 2] = y.z; k1[D / 32 - 1] = y.w;
    } else {
        const uint2 x = lds_v2(unit + g * 32 + t * 8), y = lds_v2(unit + (g + 8) * 32 + t * 8);
        k0[0] = x.x; k0[1] = x.y;
        k1[0] = y.x; k1[1] = y.y;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const uint32_t a0 = centred(k0[i] << 4), a1 = centred(k1[i] << 4), a2 = centred(k0[i]), a3 = centred(k1[i]);
        const uint32_t b0 = centred(k0[i] >> 4), b1 = centred(k1[i] >> 4), b2 = centred(k0[i] >> 8), b3 = centred(k1[i] >> 8);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            mma_16816(s[nt], a0, a1, a2, a3, q.f[nt][4 * i], q.f[nt][4 * i + 1]);
            mma_16816(s[nt], b0, b1, b2, b3, q.f[nt][4 * i + 2], q.f[nt][4 * i + 3]);
        }
    }
}

// A warp's run of units through its ring: lane u % 32 of each 32 units looks
// the unit's page up and issues its copies.
template <int D, bool kKeysOnly>
struct UnitStream {
    uint32_t ring, bars, flags;  // shared-memory addresses of this warp's slots, barriers, page-found words
    int depth, n, issued, parity, slot;
    long long u0;
    const uint8_t* src;
    bool ok;

    __device__ __forceinline__ void init(char* smem, int warp, int depth_) {
        depth = depth_;
        ring = smem_u32(smem) + warp * depth * kv_unit_bytes(D);
        bars = smem_u32(smem) + kAtWarps * depth * kv_unit_bytes(D) + warp * depth * 8;
        flags = smem_u32(smem) + kAtWarps * depth * (kv_unit_bytes(D) + 8) + warp * depth * 4;
        if ((threadIdx.x & 31) == 0)
            for (int i = 0; i < depth; ++i) mbar_init(bars + 8 * i, 1);
        fence_mbar_init();
        __syncwarp();
    }
    __device__ __forceinline__ void lookup(const KvAttendArgs& a, const Plan& p) {
        src = nullptr;
        const int i = issued + (threadIdx.x & 31);
        if (i < n) {
            const long long u = u0 + i;
            const int b = seq_of(p, a.c.n_seqs, u);
            const int ul = (p.len[b] + kKvTokens - 1) / kKvTokens;
            const long long r = u - p.pre[b];
            const int job = static_cast<int>(r / ul), ub = static_cast<int>(r - static_cast<long long>(job) * ul);
            const int h = kKeysOnly ? job : job / a.n_rt;
            const int page = kv_page(a.c, b, ub * kKvTokens);
            if (page >= 0) src = kv_unit<D>(a.c, page, h, ub * kKvTokens % a.c.page_size);
        }
    }
    // Issue the copy of the next unit of the run (every lane calls it).
    __device__ __forceinline__ void issue(const KvAttendArgs& a, const Plan& p) {
        if ((issued & 31) == 0) lookup(a, p);
        if ((threadIdx.x & 31) == (issued & 31)) {
            const int s = issued % depth;
            const uint32_t bar = bars + 8 * s, dst = ring + s * kv_unit_bytes(D);
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(flags + 4 * s), "r"(src != nullptr ? 1u : 0u) : "memory");
            if (src == nullptr) {
                mbar_arrive(bar);
            } else if (kKeysOnly) {
                mbar_arrive_expect_tx(bar, 8 * D + kKvTokens * 8);
                bulk_g2s(dst, src, 8 * D, bar);
                bulk_g2s(dst + kv_param_offset(D), src + kv_param_offset(D), kKvTokens * 8, bar);
            } else {
                mbar_arrive_expect_tx(bar, kv_unit_bytes(D));
                bulk_g2s(dst, src, kv_unit_bytes(D), bar);
            }
        }
        ++issued;
    }
    __device__ __forceinline__ void start(const KvAttendArgs& a, const Plan& p, long long first, int count) {
        u0 = first;
        n = count;
        issued = parity = slot = 0;
        ok = true;
        const int m = min(depth, n);
        for (int i = 0; i < m; ++i) issue(a, p);
    }
    // Wait for the unit in the current slot; false when the bounded wait gave up.
    __device__ __forceinline__ bool wait() {
        const bool got = mbar_wait_bounded(bars + 8 * slot, parity);
        ok = __all_sync(0xffffffffu, got);
        return ok;
    }
    __device__ __forceinline__ uint32_t unit() const { return ring + slot * kv_unit_bytes(D); }
    __device__ __forceinline__ bool found() const { return lds_u32(flags + 4 * slot) != 0; }
    // The current slot is read: refill it, go to the next.
    __device__ __forceinline__ void next(const KvAttendArgs& a, const Plan& p) {
        __syncwarp();
        if (issued < n) issue(a, p);
        if (++slot == depth) { slot = 0; parity ^= 1; }
    }
    // After a wait that gave up: no copy may still be in flight when the CTA's shared memory is released.
    __device__ __forceinline__ void drain(int consumed, unsigned int* err) {
        if ((threadIdx.x & 31) == 0) atomicOr(err, kKvErrWait);
        for (int i = consumed; i < issued; ++i) {
            mbar_wait_bounded(bars + 8 * slot, parity);
            if (++slot == depth) { slot = 0; parity ^= 1; }
        }
    }
};

// ---------------------------------------------------------------------------
// The pass over the cache
// ---------------------------------------------------------------------------
template <int D, int NT>
__global__ void __launch_bounds__(32 * kAtWarps, NT == 1 ? 4 : 3) kv_attend_kernel(const KvAttendArgs a) {
    extern __shared__ __align__(128) char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const KvView& c = a.c;
    UnitStream<D, false> st;
    st.init(smem + plan_bytes(c.n_seqs), warp, a.depth);
    pdl_launch_dependents();
    pdl_wait();
    const int warps = gridDim.x * kAtWarps;
    const Plan p = make_plan<32 * kAtWarps>(c, c.heads * a.n_rt, warps, smem, blockIdx.x == 0 ? &g_kv_attend_error : nullptr);
    const int w = warp * gridDim.x + blockIdx.x;  // neighbouring runs on different SMs
    const long long u0 = warp_start(p, w), u1 = warp_start(p, w + 1);
    const int n = static_cast<int>(u1 - u0);
    if (n == 0) return;
    st.start(a, p, u0, n);

    QueryTile<D, NT> q;
    float o[NT][D / 16][4], m[NT][2], l[NT][2], zs[NT][2], vw = 0.f;
    int b = 0, h = 0, rt = 0, len = 0, ub = 0, ul = 0, done = 0, seg = 0;
    long long left = 0;  // units of the current sequence's jobs not yet begun
    bool bad_page = false;
    while (done < n) {
        // a job, or the part of it in this run
        if (done == 0 || left == 0) {
            const long long u = u0 + done;
            b = seq_of(p, c.n_seqs, u);
            len = p.len[b];
            ul = (len + kKvTokens - 1) / kKvTokens;
            const long long r = u - p.pre[b];
            const int job = static_cast<int>(r / ul);
            ub = static_cast<int>(r - static_cast<long long>(job) * ul);
            h = job / a.n_rt;
            rt = job - h * a.n_rt;
            left = p.pre[b + 1] - u;
        }
        const int first_ub = ub, take = min(ul - ub, n - done);
        q.load(a, b, h, rt, len);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][j][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) { m[nt][e] = kNone; l[nt][e] = 0.f; zs[nt][e] = 0.f; }
        }
        vw = 2147483648.0f;  // 2^31 brings the smallest FP16 scale, 2^-24, to 2^7

        for (int i = 0; i < take; ++i, ++ub) {
            if (!st.wait()) { st.drain(done + i, &g_kv_attend_error); return; }
            const bool found = st.found();
            if (!found) bad_page = true;
            if (found && ub * kKvTokens < q.max_lim) {
                const uint32_t unit = st.unit();
                float s[NT][4];
                score_mma<D, NT>(unit, q, s);
                const uint2 p0 = lds_v2(unit + kv_param_offset(D) + 8 * g), p1 = lds_v2(unit + kv_param_offset(D) + 8 * (g + 8));
                const float sk0 = h2f_bits(lo16(p0.x)) * a.scale2, zk0 = h2f_bits(hi16(p0.x)) - 8.f;
                const float sk1 = h2f_bits(lo16(p1.x)) * a.scale2, zk1 = h2f_bits(hi16(p1.x)) - 8.f;
                float sv0 = h2f_bits(lo16(p0.y)), zv0 = h2f_bits(hi16(p0.y)) - 8.f;
                float sv1 = h2f_bits(lo16(p1.y)), zv1 = h2f_bits(hi16(p1.y)) - 8.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[nt][e] = fmaf(-zk0, q.sum[nt][e], s[nt][e]) * sk0;
                        s[nt][e + 2] = fmaf(-zk1, q.sum[nt][e], s[nt][e + 2]) * sk1;
                    }
                }
                if (ub * kKvTokens + kKvTokens > q.min_lim) {
                    // the last unit of the sequence or of a query token: keys behind a row's own are
                    // taken out, and what lies behind the last token is never multiplied
                    const int j0 = ub * kKvTokens + g, j1 = j0 + 8;
                    if (j0 >= len) { sv0 = 0.f; zv0 = 0.f; }
                    if (j1 >= len) { sv1 = 0.f; zv1 = 0.f; }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (j0 >= q.lim[nt][e]) s[nt][e] = -INFINITY;
                            if (j1 >= q.lim[nt][e]) s[nt][e + 2] = -INFINITY;
                        }
                }
                // a new maximum or a larger V scale: rare after the first units
                bool up = fmaxf(sv0, sv1) * vw > 128.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) up |= fmaxf(s[nt][e], s[nt][e + 2]) > m[nt][e] + kLazy;
                if (__any_sync(0xffffffffu, up)) {
                    const float big = lane_max_g(fmaxf(sv0, sv1));
                    float ratio = 1.f;
                    if (big * vw > 128.f) {
                        // 2^(7 - e) with 2^(e-1) <= big < 2^e
                        const float nw = __uint_as_float((260u - (__float_as_uint(big) >> 23)) << 23);
                        ratio = __uint_as_float(__float_as_uint(nw) - __float_as_uint(vw) + 0x3F800000u);  // nw / vw, powers of two
                        vw = nw;
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float top = fmaxf(m[nt][e], lane_max_g(fmaxf(s[nt][e], s[nt][e + 2])));
                            const float f = (top == m[nt][e]) ? 1.f : ex2(m[nt][e] - top);
                            m[nt][e] = top;
                            l[nt][e] *= f;
                            const float fr = f * ratio;
                            zs[nt][e] *= fr;
#pragma unroll
                            for (int j = 0; j < D / 16; ++j) { o[nt][j][e] *= fr; o[nt][j][e + 2] *= fr; }
                        }
                }
                const float w0 = sv0 * vw, w1 = sv1 * vw;
                uint32_t pf[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float e0 = ex2(s[nt][e] - m[nt][e]), e1 = ex2(s[nt][e + 2] - m[nt][e]);
                        l[nt][e] += e0 + e1;
                        x[e] = e0 * w0;
                        x[e + 2] = e1 * w1;
                        zs[nt][e] = fmaf(x[e], zv0, fmaf(x[e + 2], zv1, zs[nt][e]));
                    }
                    pf[nt][0] = movmatrix_trans(pack_f32(x[0], x[1]));
                    pf[nt][1] = movmatrix_trans(pack_f32(x[2], x[3]));
                }
                uint32_t v0[D / 32], v1[D / 32];
                const uint32_t vb = unit + kv_v_offset(D) + t * D + g * (D / 8);
                if (D == 128) {
                    const uint4 x = lds_v4(vb), y = lds_v4(vb + 4 * D);
                    v0[0] = x.x; v0[1] = x.y; v0[D / 32 - 2] = x.z; v0[D / 32 - 1] = x.w;
                    v1[0] = y.x; v1[1] = y.y; v1[D / 32 - 2] = y.z; v1[D / 32 - 1] = y.w;
                } else {
                    const uint2 x = lds_v2(vb), y = lds_v2(vb + 4 * D);
                    v0[0] = x.x; v0[1] = x.y;
                    v1[0] = y.x; v1[1] = y.y;
                }
#pragma unroll
                for (int k = 0; k < D / 32; ++k) {
                    const uint32_t a0 = centred(v0[k] << 4), a1 = centred(v0[k]), a2 = centred(v1[k] << 4), a3 = centred(v1[k]);
                    const uint32_t b0 = centred(v0[k] >> 4), b1 = centred(v0[k] >> 8), b2 = centred(v1[k] >> 4), b3 = centred(v1[k] >> 8);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_16816(o[nt][2 * k], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
                        mma_16816(o[nt][2 * k + 1], b0, b1, b2, b3, pf[nt][0], pf[nt][1]);
                    }
                }
            }
            st.next(a, p);
        }

        // the lane's columns (D/8 g ..) of rows 2t and 2t + 1
        const bool whole = first_ub == 0 && ub == ul;
        const int rows = a.tokens * a.group;
        const float inv_w = __uint_as_float(0x7F000000u - __float_as_uint(vw));  // 1 / vw, a power of two
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float ls = lane_sum_g(l[nt][e]), z = lane_sum_g(zs[nt][e]);
                const int rl = nt * 8 + 2 * t + e, r = rt * NT * 8 + rl;
                if (r >= rows) continue;
                float v[D / 8];
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    v[2 * j] = (o[nt][j][e] - z) * inv_w;
                    v[2 * j + 1] = (o[nt][j][e + 2] - z) * inv_w;
                }
                if (whole) {
                    const int tok = r / a.group, head = h * a.group + r % a.group;
                    const float f = ls > 0.f ? __fdiv_rn(1.f, ls) : (ls == 0.f ? 0.f : ls);
                    uint16_t* dst = a.out + b * a.os[0] + tok * a.os[1] + head * a.os[2] + (D / 8) * g;
#pragma unroll
                    for (int j = 0; j < D / 8; j += 8)
                        *reinterpret_cast<uint4*>(dst + j) =
                            make_uint4(pack_f32(v[j] * f, v[j + 1] * f), pack_f32(v[j + 2] * f, v[j + 3] * f),
                                       pack_f32(v[j + 4] * f, v[j + 5] * f), pack_f32(v[j + 6] * f, v[j + 7] * f));
                    if (g == 0) {
                        const size_t li = (static_cast<size_t>(b) * a.tokens + tok) * (c.heads * a.group) + head;
                        const float l2 = ls == 0.f ? -INFINITY : m[nt][e] + log2f(ls);
                        if (a.lse) a.lse[li] = l2 * 0.693147180559945309f;
                        if (a.lse2) a.lse2[li] = l2;
                    }
                } else {
                    const size_t pi = (static_cast<size_t>(w) * 2 + seg) * (NT * 8) + rl;
                    float* dst = a.part + pi * D + (D / 8) * g;
#pragma unroll
                    for (int j = 0; j < D / 8; j += 4)
                        *reinterpret_cast<float4*>(dst + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                    if (g == 0) *reinterpret_cast<float2*>(a.part_ml + pi * 2) = make_float2(m[nt][e], ls);
                }
            }
        done += take;
        left -= take;
        seg = 1;
        if (ub == ul) {
            ub = 0;
            if (++rt == a.n_rt) { rt = 0; ++h; }
        }
    }
    if (bad_page && lane == 0) atomicOr(&g_kv_attend_error, kKvErrPage);
}

// ---------------------------------------------------------------------------
// Joins the partial sums of the jobs cut between runs, in run order; writes the
// rows of sequences without keys.  One CTA per job, a warp per partial.
// ---------------------------------------------------------------------------
constexpr int kCbWarps = 8;

template <int D, int NT>
__global__ void __launch_bounds__(32 * kCbWarps) kv_combine_kernel(const KvAttendArgs a, const int warps) {
    extern __shared__ __align__(128) char smem[];
    __shared__ float so[kCbWarps][D];
    __shared__ float sml[kCbWarps][2];
    const KvView& c = a.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait();
    const Plan p = make_plan<32 * kCbWarps>(c, c.heads * a.n_rt, warps, smem, nullptr);
    const int b = blockIdx.y, job = blockIdx.x, h = job / a.n_rt, rt = job - h * a.n_rt;
    const int ul = (p.len[b] + kKvTokens - 1) / kKvTokens;
    const long long u0 = p.pre[b] + static_cast<long long>(job) * ul;
    const long long w0 = ul ? warp_of(p, u0) : 0, w1 = ul ? warp_of(p, u0 + ul - 1) : 0;
    if (ul && w0 == w1) return;  // finished by its warp
    const int rows = min(a.tokens * a.group - rt * NT * 8, NT * 8);
    const int np = ul ? static_cast<int>(w1 - w0 + 1) : 0;
    const int seg0 = ul && warp_start(p, w0) == u0 ? 0 : 1;
    constexpr int V = D / 32;  // columns of a lane
    for (int rl = 0; rl < rows; ++rl) {
        float m = kNone, l = 0.f, o[V];
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = 0.f;
        for (int i = warp; i < np; i += kCbWarps) {
            const size_t pi = (static_cast<size_t>(w0 + i) * 2 + (i == 0 ? seg0 : 0)) * (NT * 8) + rl;
            const float mi = ldcg_f32(a.part_ml + 2 * pi), li = ldcg_f32(a.part_ml + 2 * pi + 1);
            const float top = fmaxf(m, mi), f0 = ex2(m - top), f1 = ex2(mi - top);
            m = top;
            l = l * f0 + li * f1;
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = o[k] * f0 + ldcg_f32(a.part + pi * D + lane + 32 * k) * f1;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; ++k) so[warp][lane + 32 * k] = o[k];
        if (lane == 0) { sml[warp][0] = m; sml[warp][1] = l; }
        __syncthreads();
        const int r = rt * NT * 8 + rl, tok = r / a.group, head = h * a.group + r % a.group;
        if (tid < D) {
            float top = kNone;
#pragma unroll
            for (int i = 0; i < kCbWarps; ++i) top = fmaxf(top, sml[i][0]);
            float ls = 0.f, v = 0.f;
#pragma unroll
            for (int i = 0; i < kCbWarps; ++i) {
                const float f = ex2(sml[i][0] - top);
                ls += sml[i][1] * f;
                v += so[i][tid] * f;
            }
            const float f = ls > 0.f ? __fdiv_rn(1.f, ls) : (ls == 0.f ? 0.f : ls);
            a.out[b * a.os[0] + tok * a.os[1] + head * a.os[2] + tid] = __half_as_ushort(__float2half_rn(v * f));
            if (tid == 0) {
                const size_t li = (static_cast<size_t>(b) * a.tokens + tok) * (c.heads * a.group) + head;
                const float l2 = ls == 0.f ? -INFINITY : top + log2f(ls);
                if (a.lse) a.lse[li] = l2 * 0.693147180559945309f;
                if (a.lse2) a.lse2[li] = l2;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Accumulated weight: mass_j += sum over the rows of exp2(score - lse), a second
// pass over the keys alone (8 D + 128 of a unit's 16 D + 128 bytes) now that
// every row's lse is known.  A slot's sum is one lane group's, in row order.
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(32 * kAtWarps, 4) kv_mass_kernel(const KvAttendArgs a) {
    extern __shared__ __align__(128) char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const KvView& c = a.c;
    UnitStream<D, true> st;
    st.init(smem + plan_bytes(c.n_seqs), warp, a.depth);
    pdl_launch_dependents();
    pdl_wait();
    const Plan p = make_plan<32 * kAtWarps>(c, c.heads, gridDim.x * kAtWarps, smem, nullptr);
    const int w = warp * gridDim.x + blockIdx.x;
    const long long u0 = warp_start(p, w);
    const int n = static_cast<int>(warp_start(p, w + 1) - u0);
    if (n == 0) return;
    st.start(a, p, u0, n);
    QueryTile<D, 1> q;
    const int n_rt = (a.tokens * a.group + 7) / 8, rows = a.tokens * a.group;
    int last_b = -1, last_h = -1;
    float lse[2] = {0.f, 0.f};
    for (int i = 0; i < n; ++i) {
        const long long u = u0 + i;
        const int b = seq_of(p, c.n_seqs, u), len = p.len[b], ul = (len + kKvTokens - 1) / kKvTokens;
        const long long r = u - p.pre[b];
        const int h = static_cast<int>(r / ul), ub = static_cast<int>(r - static_cast<long long>(h) * ul);
        if (!st.wait()) { st.drain(i, &g_kv_attend_error); return; }
        if (st.found()) {
            const uint32_t unit = st.unit();
            const uint2 p0 = lds_v2(unit + kv_param_offset(D) + 8 * g), p1 = lds_v2(unit + kv_param_offset(D) + 8 * (g + 8));
            const float sk0 = h2f_bits(lo16(p0.x)) * a.scale2, zk0 = h2f_bits(hi16(p0.x)) - 8.f;
            const float sk1 = h2f_bits(lo16(p1.x)) * a.scale2, zk1 = h2f_bits(hi16(p1.x)) - 8.f;
            const int j0 = ub * kKvTokens + g, j1 = j0 + 8;
            float add0 = 0.f, add1 = 0.f;
            for (int rt = 0; rt < n_rt; ++rt) {
                if (n_rt > 1 || b != last_b || h != last_h) {
                    q.load(a, b, h, rt, len);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int row = rt * 8 + 2 * t + e;
                        lse[e] = INFINITY;  // padding rows weigh nothing
                        if (row < rows) {
                            const int tok = row / a.group, head = h * a.group + row % a.group;
                            lse[e] = ldcg_f32(a.lse2 + (static_cast<size_t>(b) * a.tokens + tok) * (c.heads * a.group) + head);
                            if (lse[e] == -INFINITY) lse[e] = INFINITY;  // a row without keys
                        }
                    }
                    last_b = b;
                    last_h = h;
                }
                if (ub * kKvTokens >= q.max_lim) continue;
                float s[1][4];
                score_mma<D, 1>(unit, q, s);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float e0 = ex2(fmaf(-zk0, q.sum[0][e], s[0][e]) * sk0 - lse[e]);
                    const float e1 = ex2(fmaf(-zk1, q.sum[0][e], s[0][e + 2]) * sk1 - lse[e]);
                    if (j0 < q.lim[0][e]) add0 += e0;
                    if (j1 < q.lim[0][e]) add1 += e1;
                }
            }
            add0 += __shfl_xor_sync(0xffffffffu, add0, 1);
            add1 += __shfl_xor_sync(0xffffffffu, add1, 1);
            add0 += __shfl_xor_sync(0xffffffffu, add0, 2);
            add1 += __shfl_xor_sync(0xffffffffu, add1, 2);
            const int page = kv_page(c, b, ub * kKvTokens);
            if (page >= 0 && t < 2) {
                const int j = t == 0 ? j0 : j1;
                if (j < len) c.mass[kv_line(c, page, h) + j % c.page_size] += t == 0 ? add0 : add1;
            }
        }
        st.next(a, p);
    }
}

constexpr int kAtSmemPerSm = 226 * 1024;

// Shared memory of a CTA when `ctas` of them share an SM, and the ring depth that fits.
int ring_depth(int n_seqs, int d, int ctas, int* smem) {
    const int room = kAtSmemPerSm / ctas - 1024 - plan_bytes(n_seqs) - 256;
    int depth = room / (kAtWarps * (kv_unit_bytes(d) + 12));
    depth = depth > 12 ? 12 : depth;
    *smem = plan_bytes(n_seqs) + (kAtWarps * depth * (kv_unit_bytes(d) + 12) + 127) / 128 * 128;
    return depth;
}

template <class K>
dq_status_t allow_smem(K kernel, int smem) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { set_cuda_error(e); return DQ_ERR_CUDA; }
    return DQ_OK;
}

template <int D, int NT>
dq_status_t attend(KvAttendArgs& a, cudaStream_t stream) {
    DeviceInfo di;
    dq_status_t st = device_info(&di);
    if (st != DQ_OK) return st;
    const int ctas = NT == 1 ? 4 : 3;
    int grid = di.sm_count * ctas;
    if (grid * kAtWarps > kAtMaxWarps) grid = kAtMaxWarps / kAtWarps;
    int smem = 0;
    a.depth = ring_depth(a.c.n_seqs, D, ctas, &smem);
    if ((st = allow_smem(kv_attend_kernel<D, NT>, smem)) != DQ_OK) return st;
    if ((st = launch_pdl(kv_attend_kernel<D, NT>, dim3(grid), 32 * kAtWarps, smem, stream, a)) != DQ_OK) return st;
    const dim3 jobs(a.c.heads * a.n_rt, a.c.n_seqs);
    st = launch_pdl(kv_combine_kernel<D, NT>, jobs, 32 * kCbWarps, plan_bytes(a.c.n_seqs), stream, a, grid * kAtWarps);
    if (st != DQ_OK || !a.lse2) return st;
    grid = di.sm_count * 4;
    if (grid * kAtWarps > kAtMaxWarps) grid = kAtMaxWarps / kAtWarps;
    a.depth = ring_depth(a.c.n_seqs, D, 4, &smem);
    if ((st = allow_smem(kv_mass_kernel<D>, smem)) != DQ_OK) return st;
    return launch_pdl(kv_mass_kernel<D>, dim3(grid), 32 * kAtWarps, smem, stream, a);
}

// Row tiles of one warp: 8 rows when a KV head has no more, else 16.
int row_tiles(int rows) { return rows <= 8 ? 1 : 2; }

struct AttendWs {
    size_t part, ml, lse2, total;
};
AttendWs attend_ws(const dq_kv_cache_t& c, int tokens, int q_heads, bool mass) {
    const int nt = row_tiles(tokens * (q_heads / c.kv_heads));
    const size_t rows = static_cast<size_t>(kAtMaxWarps) * 2 * 8 * nt;
    AttendWs w;
    w.part = 0;
    w.ml = align256(rows * c.head_dim * 4);
    w.lse2 = w.ml + align256(rows * 8);
    w.total = w.lse2 + (mass ? align256(static_cast<size_t>(c.n_seqs) * tokens * q_heads * 4) : 0);
    return w;
}

}  // namespace

size_t kv_attend_workspace(const dq_kv_cache_t& c, int tokens, int q_heads, bool mass) {
    return attend_ws(c, tokens, q_heads, mass).total;
}

dq_status_t launch_kv_attend(const dq_kv_cache_t& c, const dq_kv_attend_t& r, void* workspace, cudaStream_t stream) {
    KvAttendArgs a{};
    a.c = kv_view(c);
    a.q = r.q;
    a.out = r.out;
    for (int i = 0; i < 3; ++i) { a.qs[i] = r.q_stride[i]; a.os[i] = r.out_stride[i]; }
    a.lse = r.lse;
    a.counts = r.counts;
    a.tokens = r.tokens;
    a.group = r.q_heads / c.kv_heads;
    a.scale2 = r.scale * 1.44269504088896341f;
    const AttendWs w = attend_ws(c, r.tokens, r.q_heads, r.accumulate != 0);
    char* base = static_cast<char*>(workspace);
    a.part = reinterpret_cast<float*>(base + w.part);
    a.part_ml = reinterpret_cast<float*>(base + w.ml);
    a.lse2 = r.accumulate ? reinterpret_cast<float*>(base + w.lse2) : nullptr;
    const int rows = r.tokens * a.group, nt = row_tiles(rows);
    a.n_rt = (rows + 8 * nt - 1) / (8 * nt);
    if (c.head_dim == 128) return nt == 1 ? attend<128, 1>(a, stream) : attend<128, 2>(a, stream);
    return nt == 1 ? attend<64, 1>(a, stream) : attend<64, 2>(a, stream);
}

dq_status_t read_kv_attend_error(uint32_t* word, bool clear) {
    unsigned int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_kv_attend_error, sizeof(v));
    if (e == cudaSuccess && clear && v) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_kv_attend_error, &zero, sizeof(zero));
    }
    if (e != cudaSuccess) { set_cuda_error(e); return DQ_ERR_CUDA; }
    *word = v;
    return DQ_OK;
}

}  // namespace dq
