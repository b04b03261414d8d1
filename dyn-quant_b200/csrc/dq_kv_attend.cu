// dq_kv_attend.cu -- attention of the newest tokens over the paged 4-bit KV
// cache (layout in dq_kv.cuh).  No counterpart in the reference.
//
//   out_r = sum_j p_rj V_j,  p_rj = softmax_j(scale <q_r, K_j>),  K_j = s_j (c_j - z_j), V_j alike
//
// One pass over the cache with the running maximum and sum of the softmax.
// Rows r = (query token, query head of the KV head) share the KV head's units.
//
// Work split: the steps (32 slots, two units) of all (sequence, KV head, row
// tile) jobs form one list, cut into equal runs, one per warp of a persistent
// grid, so ragged lengths, few sequences and long ones all fill the GPU.  Each
// warp streams its run through a ring of bulk copies of its own; job borders do
// not interrupt the stream.  A job inside one run is finished there.  The pieces
// of the others meet in shared memory when their CTA's warps (neighbouring
// runs) are done.  What a CTA's border still cuts leaves its partial sums
// (maximum, sum, unnormalised output) in the workspace, and the last of the
// job's CTAs to arrive joins them (for several row tiles, kv_combine_kernel
// does).  All sums have a fixed order.
//
// Products (mma.sync.m16n8k16, f16 x f16 -> f32) are transposed, so that the 16
// slots of a unit are the MMA's rows and the query rows its 8 columns:
//   S^T = K Q^T    A = 16 slots x 16 columns of K, B = Q^T
//   O^T = V^T P^T A = 16 columns of V x 16 slots, B = P^T
// A decode step has at most 8 rows per KV head, so nothing of an MMA is idle,
// and a lane's S values (slots g, g + 8; rows 2t, 2t + 1) lie in the lanes that
// hold its O columns' rows: maxima, sums and rescaling stay in the lane.
// A nibble at bits 0..3 or 4..7 of a half word is the subnormal f16 number c 2^-24
// or c 2^-20, which an MMA multiplies exactly, so a word of eight codes costs one
// shift and four masks.  But an MMA cuts its terms off below the largest, for which
// a subnormal counts as 2^-14.  Scores are not to feel that (with one column of q at
// 4000 and the rest below 1 they were off by 0.5 in units of a code, 200 times what
// normal numbers give): keys are brought to c 2^-14 by one multiplication a pair
// (64 sequences of 2000 to 4096 slots with 32 heads: 166 -> 171.5 us; 131071 slots
// with 8 heads of 8 rows: 46.0 -> 46.9).  In the output the values' codes are used as they
// lie: the two weights lie in different rows of the MMA and are set right at the
// end.  Scales and zeros are applied in FP32:
//   S   = s_k (D - z_k sum q),  D the MMAs' sum of q c
//   O   = sum p' (c - 8) - sum p' (z_v - 8),  p' = p s_v w
// The 8 is the same for all columns: one MMA a unit with a constant A collects
// 8 sum p' and every 8 steps it is taken off all of O, which keeps the running
// sums (FP32, and the rounding of p' in them) at the size of the centred values.
// Codes all have one sign, so what is cut off adds up: the output of 128K slots, a
// thousandth of a value's size, leaned by 2e-4 of it.  So the second unit of a step
// is taken the other way round, -p' with 15 - c, and the errors cancel (1% of the time).
// p' is the only rounding to FP16 besides the output's: p <= 2^8 (the maximum
// is taken again only when a score passes it by 8) and w is the power of two
// that brings the largest s_v seen to at most 2^7, so p' <= 2^15.  Weights keep their
// 11 bits down to about 2^-20 of the largest (p' of 2^-14, where that has 2^6 to 2^7;
// 2^-28 where the maximum lags by its 8), below it they lose one a halving.
//
// Measured: 64 sequences of 2000 to 4096 slots with 32 heads of 128 and one row
// each, 850 MB, 171 to 183 us, 4.6 to 5.0 TB/s (72 to 77% of a copy's; 59% of the
// issue slots, the tensor pipe 30%); 16 sequences of 1000 to 4100 slots with 8
// heads of 8 rows, 48 MB, 26 us; 131071 slots with 8 heads of 8 rows, 143 MB, 47
// us; 8 sequences of 200 to 8000 slots with 8 heads of 64 and 20 rows, 22 MB, 38
// us with the join.  The smaller ones are bound by the chain lengths, pages, units,
// join: 77 slots of 32 heads take 9.2 us.
#include "dq_kv_plan.cuh"

namespace dq {

namespace {

__device__ unsigned int g_kv_attend_error;

constexpr int kAtMaxWarps = 2560;     // bound on the grid's warps (workspace sizing)
constexpr float kCode = 16777216.0f;  // 2^24: a masked low code is c / kCode
constexpr float kKey = 16384.0f;      // 2^14: a key's code in its product is c / kKey

// Warps of a CTA and CTAs of an SM for row tiles of 8 NT rows: with one tile a thread
// has 128 registers, with two 168, of which heads of 128 spill some 250 bytes.
__host__ __device__ constexpr int at_warps(int nt) { return nt == 1 ? 8 : 10; }
__host__ __device__ constexpr int at_ctas(int nt) { return nt == 1 ? 2 : 1; }

// f16 pairs c 2^-24 of the nibbles at bits 0..3 and 16..19, c 2^-20 of those at bits 4..7 and 20..23.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return w & 0x000F000Fu; }
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return w & 0x00F000F0u; }
// Both as c 2^-14, normal numbers (exact).
__device__ __forceinline__ uint32_t times(uint32_t w, uint32_t pow2) {
    uint32_t r;
    asm("mul.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(pow2));
    return r;
}
__device__ __forceinline__ uint32_t low_keys(uint32_t w) { return times(low_codes(w), 0x64006400u); }
__device__ __forceinline__ uint32_t high_keys(uint32_t w) { return times(high_codes(w), 0x54005400u); }
// mask & ~w, the codes 15 - c, in one instruction (left to itself, ~w would be one of its own)
__device__ __forceinline__ uint32_t and_not(uint32_t mask, uint32_t w) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %1, 0x30;" : "=r"(r) : "r"(mask), "r"(w));
    return r;
}

// mma_16816 that the compiler may move (it has no effect besides its result).
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Dynamic shared memory by its byte offset.
template <class T>
__device__ __forceinline__ T smem_at(int off) {
    extern __shared__ __align__(128) char smem[];
    return *reinterpret_cast<const T*>(smem + off);
}

// D/32 words at once: 16 or 8 bytes.
template <int D>
__device__ __forceinline__ void load_words(int off, uint32_t (&w)[D / 32]) {
    if (D == 128) {
        const uint4 x = smem_at<uint4>(off);
        w[0] = x.x; w[1] = x.y; w[D / 32 - 2] = x.z; w[D / 32 - 1] = x.w;
    } else {
        const uint2 x = smem_at<uint2>(off);
        w[0] = x.x; w[1] = x.y;
    }
}

// An 8x8 matrix of b16 in the MMA layout, transposed across the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
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
    f2 sum[NT];             // - sum of q over the columns / kKey, rows 2t and 2t + 1
    int lim[NT][2];         // keys that rows 2t and 2t + 1 see
    int min_lim, max_lim;   // over the tile's rows

    int cnt;
    // Request row r of the job, query token r / group, head h * group + r % group, ...
    __device__ __forceinline__ void request(const KvAttendArgs& a, int b, int h, int rt, uint4 (&raw)[NT][D / 32]) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const int rows = a.tokens * a.group;
        cnt = a.counts ? min(max(ld_l2(a.counts + b), 0), a.tokens) : a.tokens;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = (rt * NT + nt) * 8 + g, tok = r / a.group;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                raw[nt][i] = make_uint4(0, 0, 0, 0);
                if (r < rows && tok < cnt)
                    raw[nt][i] = ld_l2_v4(a.q + b * a.qs[0] + tok * a.qs[1] + (h * a.group + r - tok * a.group) * a.qs[2] + (D / 4) * t + 8 * i);
            }
        }
    }
    // ... and arrange it.
    __device__ __forceinline__ void arrange(const KvAttendArgs& a, int rt, int len, const uint4 (&raw)[NT][D / 32]) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const int rows = a.tokens * a.group;
        int lo = len, hi = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = (rt * NT + nt) * 8 + g, tok = r / a.group;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const uint4 w = raw[nt][i];
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
            s *= -1.f / kKey;
            sum[nt] = f2(__shfl_sync(0xffffffffu, s, 8 * t), __shfl_sync(0xffffffffu, s, 8 * t + 4));
#pragma unroll
            for (int e = 0; e < 2; ++e) lim[nt][e] = __shfl_sync(0xffffffffu, l, 8 * t + 4 * e);
        }
        min_lim = __reduce_min_sync(0xffffffffu, lo);
        max_lim = __reduce_max_sync(0xffffffffu, hi);
    }
    __device__ __forceinline__ void load(const KvAttendArgs& a, int b, int h, int rt, int len) {
        uint4 raw[NT][D / 32];
        request(a, b, h, rt, raw);
        arrange(a, rt, len, raw);
    }
};

// D / kKey of U units, D the MMAs' sums of q c for slots g, g + 8 and rows 2t, 2t + 1.
template <int D, int NT, int U>
__device__ __forceinline__ void score_mma(int unit, const QueryTile<D, NT>& q, f2 (&s)[U][NT][2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t k0[U][D / 32], k1[U][D / 32];
    float lo[U][NT][4], hi[U][NT][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int at = unit + u * kv_unit_bytes(D) + g * (D / 2) + t * (D / 8);
        load_words<D>(at, k0[u]);
        load_words<D>(at + 8 * (D / 2), k1[u]);
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t w0 = k0[u][i], w1 = k1[u][i], x0 = w0 >> 8, x1 = w1 >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (i == 0) {
                    mma_first(lo[u][nt], low_keys(w0), low_keys(w1), low_keys(x0), low_keys(x1), q.f[nt][0], q.f[nt][2]);
                    mma_first(hi[u][nt], high_keys(w0), high_keys(w1), high_keys(x0), high_keys(x1), q.f[nt][1], q.f[nt][3]);
                } else {
                    mma(lo[u][nt], low_keys(w0), low_keys(w1), low_keys(x0), low_keys(x1), q.f[nt][4 * i], q.f[nt][4 * i + 2]);
                    mma(hi[u][nt], high_keys(w0), high_keys(w1), high_keys(x0), high_keys(x1), q.f[nt][4 * i + 1],
                        q.f[nt][4 * i + 3]);
                }
            }
        }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                s[u][nt][x] = f2(hi[u][nt][2 * x], hi[u][nt][2 * x + 1]) + f2(lo[u][nt][2 * x], lo[u][nt][2 * x + 1]);
}

// A warp's run of steps through its ring: lane i % 32 of each 32 steps looks
// the step's pages up and issues its copies.
template <int D>
struct StepStream {
    static constexpr int kUnit = kv_unit_bytes(D);
    static constexpr int kSlot = 2 * kUnit;
    int ring, bars, units;       // offsets in shared memory of this warp's slots, barriers, the slots' unit indices
    int depth, n, issued, parity, slot;
    bool absent;                 // some unit of the run lies in no page of the pool
    long long u0;
    int src[2];                  // this lane's step: the units' indices in the pool, -1: none

    // Bytes of `warps` rings behind `smem`.
    static __host__ __device__ int bytes(int warps, int depth) { return (warps * depth * (kSlot + 16) + 127) / 128 * 128; }

    static __device__ __forceinline__ uint32_t base() {
        extern __shared__ __align__(128) char smem[];
        return smem_u32(smem);
    }
    __device__ __forceinline__ void init(int off, int warps, int warp, int depth_) {
        depth = depth_;
        ring = off + warp * depth * kSlot;
        bars = off + warps * depth * kSlot + warp * depth * 8;
        units = off + warps * depth * (kSlot + 8) + warp * depth * 8;
        if ((threadIdx.x & 31) == 0)
            for (int i = 0; i < depth; ++i) mbar_init(base() + bars + 8 * i, 1);
        fence_mbar_init();
        __syncwarp();
    }
    __device__ __forceinline__ StepAt lookup(const KvAttendArgs& a, const Plan& p) {
        src[0] = src[1] = -1;
        bool bad = false;
        const int i = issued + (threadIdx.x & 31);
        StepAt x{0, 0, 0, 0};
        if (i < n) {
            x = step_at(p, a.c.n_seqs, u0 + i);
            const int h = x.job / a.n_rt;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int s = x.step * kStep + e * kKvTokens;
                if (s >= x.len) break;
                const int page = kv_page(a.c, x.b, s);
                if (page >= 0) src[e] = static_cast<int>((kv_line(a.c, page, h) + s % a.c.page_size) / kKvTokens);
                else bad = true;
            }
        }
        if (__any_sync(0xffffffffu, bad)) absent = true;
        return x;
    }
    // Issue the copies of the run's next step into slot s (every lane calls it).
    __device__ __forceinline__ void issue(const KvAttendArgs& a, const Plan& p, int s) {
        if (issued > 0 && (issued & 31) == 0) lookup(a, p);
        const int i0 = __shfl_sync(0xffffffffu, src[0], issued), i1 = __shfl_sync(0xffffffffu, src[1], issued);
        if ((threadIdx.x & 31) == 0) {
            const uint32_t bar = base() + bars + 8 * s, dst = base() + ring + s * kSlot;
            asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(base() + units + 8 * s), "r"(i0), "r"(i1) : "memory");
            if (i0 >= 0 && i1 == i0 + 1) {
                mbar_arrive_expect_tx(bar, kSlot);
                bulk_g2s(dst, a.c.units + static_cast<size_t>(i0) * kUnit, kSlot, bar);
            } else {
                issue_units(a, bar, dst, i0, i1);
            }
        }
        ++issued;
    }
    // A step's units one by one: from different pages, or one of them missing.
    __device__ __forceinline__ void issue_units(const KvAttendArgs& a, uint32_t bar, uint32_t dst, int i0, int i1) {
        if (i0 < 0 && i1 < 0) {
            mbar_arrive(bar);
            return;
        }
        mbar_arrive_expect_tx(bar, (i0 >= 0 ? kUnit : 0) + (i1 >= 0 ? kUnit : 0));
        if (i0 >= 0) bulk_g2s(dst, a.c.units + static_cast<size_t>(i0) * kUnit, kUnit, bar);
        if (i1 >= 0) bulk_g2s(dst + kUnit, a.c.units + static_cast<size_t>(i1) * kUnit, kUnit, bar);
    }
    // Where the run begins; then fill() asks for its first steps.
    __device__ __forceinline__ StepAt start(const KvAttendArgs& a, const Plan& p, long long first, int count) {
        u0 = first;
        n = count;
        issued = parity = slot = 0;
        absent = false;
        StepAt x = lookup(a, p);
        x.b = __shfl_sync(0xffffffffu, x.b, 0);
        x.len = __shfl_sync(0xffffffffu, x.len, 0);
        x.job = __shfl_sync(0xffffffffu, x.job, 0);
        x.step = __shfl_sync(0xffffffffu, x.step, 0);
        return x;
    }
    __device__ __forceinline__ void fill(const KvAttendArgs& a, const Plan& p) {
        const int m = min(depth, n);
        for (int i = 0; i < m; ++i) issue(a, p, i);
    }
    // Wait for the step's copies; false when the bounded wait gave up.
    __device__ __forceinline__ bool wait() {
        return __all_sync(0xffffffffu, mbar_wait_bounded(base() + bars + 8 * slot, parity));
    }
    __device__ __forceinline__ int unit() const { return ring + slot * kSlot; }
    // The step's units in the pool, -1: not copied.
    __device__ __forceinline__ int2 unit_index() const { return smem_at<int2>(units + 8 * slot); }
    // Bit e: unit e of the step was copied (only asked for when some unit of the run is absent).
    __device__ __forceinline__ uint32_t found() const {
        const int2 i = unit_index();
        return (i.x >= 0 ? 1u : 0u) | (i.y >= 0 ? 2u : 0u);
    }
    // The current slot is read: refill it, go to the next.
    __device__ __forceinline__ void next(const KvAttendArgs& a, const Plan& p) {
        __syncwarp();
        if (issued < n) issue(a, p, slot);
        if (++slot == depth) { slot = 0; parity ^= 1; }
    }
    // After a wait that gave up: no copy may still be in flight when the CTA's shared memory is released.
    __device__ __forceinline__ void drain(int consumed) {
        if ((threadIdx.x & 31) == 0) atomicOr(&g_kv_attend_error, kKvErrWait);
        for (int i = consumed; i < issued; ++i) {
            mbar_wait_bounded(base() + bars + 8 * slot, parity);
            if (++slot == depth) { slot = 0; parity ^= 1; }
        }
    }
};

// The running softmax of one job in one warp: rows 2t, 2t + 1 of each row tile.
template <int D, int NT>
struct RowState {
    float o[NT][D / 16][4], c8[NT][4], vw;  // c8: -+ 8 sum p' since the last settle(), in either scale of o
    f2 m[NT], l[NT], zs[NT];  // m: minus the running maximum

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][j][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) c8[nt][e] = 0.f;
            m[nt] = f2(-kNone);
            l[nt] = zs[nt] = f2(0.f);
        }
        vw = 2147483648.0f;  // 2^31 brings the smallest FP16 scale, 2^-24, to 2^7
    }

    // Scores and weights of U units from slot j of the sequence on, the weights as the B operands of their
    // output product, and the units' V codes.  found: bit u set where unit u is there.  kFirst: the first unit's
    // place in its step.
    template <int U, int kFirst, bool kScores>
    __device__ __forceinline__ void weigh(const QueryTile<D, NT>& q, int unit, int j, int len, uint32_t found, float scale2,
                                          uint32_t (&pf)[U][NT][2], uint32_t (&v)[U][2][D / 32], float* scores, int pitch,
                                          int2 index) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        f2 s[U][NT][2];
        float sv[U][2], zv[U][2];
        score_mma<D, NT, U>(unit, q, s);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int pa = unit + u * kv_unit_bytes(D) + kv_param_offset(D) + 8 * g;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint2 p = smem_at<uint2>(pa + 64 * x);
                const f2 sk(h2f_bits(lo16(p.x)) * scale2), zk(h2f_bits(hi16(p.x)));
                sv[u][x] = h2f_bits(lo16(p.y));
                // -p' (15 - c) + 8 p' - p' = p' (c - 8)
                zv[u][x] = (u + kFirst) % 2 ? 7.f - h2f_bits(hi16(p.y)) : h2f_bits(hi16(p.y)) - 8.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[u][nt][x] = fma2(zk, q.sum[nt], s[u][nt][x]) * sk;
            }
        }
        if (j + U * kKvTokens > q.min_lim || found != (1u << U) - 1u) {
            // the end of the sequence or of a query token's keys, or an absent page: slots behind a
            // row's keys are taken out, and what lies behind the last token is never multiplied
            bool odd = false;
#pragma unroll
            for (int u = 0; u < U; ++u) odd |= !(fabsf(sv[u][0]) + fabsf(sv[u][1]) + fabsf(zv[u][0]) + fabsf(zv[u][1]) < INFINITY);
            if (__any_sync(0xffffffffu, odd)) {
                // a value row that is not finite (or is not there): the outputs of the rows that see it are not either,
                // and it must not meet the zero weights of those that do not
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int jj = j + u * kKvTokens + g + 8 * x;
                        if (fabsf(sv[u][x]) + fabsf(zv[u][x]) < INFINITY) continue;
                        const bool there = jj < len && (found >> u & 1u);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            zs[nt] = zs[nt] + f2(there && jj < q.lim[nt][0] ? NAN : 0.f, there && jj < q.lim[nt][1] ? NAN : 0.f);
                        sv[u][x] = 0.f;
                        zv[u][x] = 0.f;
                    }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int jj = j + u * kKvTokens + g + 8 * x;
                    const bool there = jj < len && (found >> u & 1u);
                    if (!there) { sv[u][x] = 0.f; zv[u][x] = 0.f; }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        s[u][nt][x] = f2(there && jj < q.lim[nt][0] ? s[u][nt][x].x() : -INFINITY,
                                         there && jj < q.lim[nt][1] ? s[u][nt][x].y() : -INFINITY);
                }
        }
        if (kScores) {
            // kept for the mass pass: [unit][slot][pitch], the lane's rows 2t, 2t + 1
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = u ? index.y : index.x;
                if (i < 0 || 2 * t >= pitch) continue;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float* dst = scores + (static_cast<size_t>(i) * kKvTokens + g + 8 * x) * pitch + 2 * t;
                    if (pitch == 1) *dst = s[u][0][x].x();
                    else *reinterpret_cast<float2*>(dst) = make_float2(s[u][0][x].x(), s[u][0][x].y());
                }
            }
        }
        // a new maximum or a larger V scale: rare after the first steps
        float big = fmaxf(sv[0][0], sv[0][1]), top[NT][2];
#pragma unroll
        for (int u = 1; u < U; ++u) big = fmaxf(big, fmaxf(sv[u][0], sv[u][1]));
        bool up = big * vw > 128.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            top[nt][0] = fmaxf(s[0][nt][0].x(), s[0][nt][1].x());
            top[nt][1] = fmaxf(s[0][nt][0].y(), s[0][nt][1].y());
#pragma unroll
            for (int u = 1; u < U; ++u) {
                top[nt][0] = fmaxf(top[nt][0], fmaxf(s[u][nt][0].x(), s[u][nt][1].x()));
                top[nt][1] = fmaxf(top[nt][1], fmaxf(s[u][nt][0].y(), s[u][nt][1].y()));
            }
            up |= top[nt][0] + m[nt].x() > kLazy;
            up |= top[nt][1] + m[nt].y() > kLazy;
        }
        if (__any_sync(0xffffffffu, up)) rescale(top, big);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int vb = unit + u * kv_unit_bytes(D) + kv_v_offset(D) + t * D + g * (D / 8);
            load_words<D>(vb, v[u][0]);
            load_words<D>(vb + 4 * D, v[u][1]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const f2 w((u + kFirst) % 2 ? -(sv[u][x] * vw) : sv[u][x] * vw), z(zv[u][x]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const f2 d = s[u][nt][x] + m[nt], e(ex2(d.x()), ex2(d.y())), p = e * w;
                    l[nt] = l[nt] + e;
                    zs[nt] = fma2(p, z, zs[nt]);
                    pf[u][nt][x] = movmatrix_trans(pack_f32(p.x(), p.y()));
                }
            }
    }

    // The output product of what weigh() left.  Rows g of an MMA are columns of low nibbles, rows g + 8 of
    // high ones; the constants are -8 in either.
    template <int U, int kFirst>
    __device__ __forceinline__ void output(const uint32_t (&pf)[U][NT][2], const uint32_t (&v)[U][2][D / 32]) {
        constexpr uint32_t kLow8 = 0x80088008u, kHigh8 = 0x80808080u;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            auto lows = [&](uint32_t w) { return (u + kFirst) % 2 ? and_not(0x000F000Fu, w) : low_codes(w); };
            auto highs = [&](uint32_t w) { return (u + kFirst) % 2 ? and_not(0x00F000F0u, w) : high_codes(w); };
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma(c8[nt], kLow8, kHigh8, kLow8, kHigh8, pf[u][nt][0], pf[u][nt][1]);
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                const uint32_t w0 = v[u][0][k], w1 = v[u][1][k], y0 = w0 >> 8, y1 = w1 >> 8;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t b0 = pf[u][nt][0], b1 = pf[u][nt][1];
                    mma(o[nt][2 * k], lows(w0), highs(w0), lows(w1), highs(w1), b0, b1);
                    mma(o[nt][2 * k + 1], lows(y0), highs(y0), lows(y1), highs(y1), b0, b1);
                }
            }
        }
    }

    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) o[nt][k][x] += c8[nt][x];
                c8[nt][x] = 0.f;
            }
    }

    __device__ __forceinline__ void rescale(const float (&top)[NT][2], float big) {
        big = lane_max_g(big);
        float ratio = 1.f;
        if (big * vw > 128.f) {
            // 2^(7 - e) with 2^(e-1) <= big < 2^e
            const float nw = __uint_as_float((260u - (__float_as_uint(big) >> 23)) << 23);
            ratio = __uint_as_float(__float_as_uint(nw) - __float_as_uint(vw) + 0x3F800000u);  // nw / vw, powers of two
            vw = nw;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float now[2], f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float old = -(e ? m[nt].y() : m[nt].x());
                now[e] = fmaxf(old, lane_max_g(top[nt][e]));
                f[e] = (now[e] == old) ? 1.f : ex2(old - now[e]);
            }
            m[nt] = f2(-now[0], -now[1]);
            l[nt] = l[nt] * f2(f[0], f[1]);
            const f2 fr(f[0] * ratio, f[1] * ratio);
            zs[nt] = zs[nt] * fr;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[nt][k][x] *= (x & 1) ? fr.y() : fr.x();
#pragma unroll
            for (int x = 0; x < 4; ++x) c8[nt][x] *= (x & 1) ? fr.y() : fr.x();
        }
    }

    // Row 2t + e of tile nt: its sum of weights and the lane's columns D/8 g .. of its unnormalised output.
    __device__ __forceinline__ float finish(int nt, int e, float (&v)[D / 8]) const {
        const float z = lane_sum_g(e ? zs[nt].y() : zs[nt].x());
        const float inv = __uint_as_float(0x7F000000u - __float_as_uint(vw));  // 1 / vw
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            v[2 * k] = fmaf(o[nt][k][e], kCode, -z) * inv;
            v[2 * k + 1] = fmaf(o[nt][k][e + 2], kCode / 16.f, -z) * inv;
        }
        return lane_sum_g(e ? l[nt].y() : l[nt].x());
    }
    __device__ __forceinline__ float top(int nt, int e) const { return -(e ? m[nt].y() : m[nt].x()); }
};

// A piece of a job that its run cut: which job and which of its steps.
struct Piece {
    int b, job, first, end;  // job < 0: none
};

// ---------------------------------------------------------------------------
// The pass over the cache
// ---------------------------------------------------------------------------
template <int D, int NT, bool kScores>
__global__ void __launch_bounds__(32 * at_warps(NT), at_ctas(NT)) kv_attend_kernel(const KvAttendArgs a) {
    constexpr int W = at_warps(NT), R = 8 * NT;
    static_assert(2 * W <= 32, "a lane per piece");
    extern __shared__ __align__(128) char smem[];
    __shared__ Piece pieces[2 * W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const KvView& c = a.c;
    __shared__ Piece cut[2];
    __shared__ Share share[2];
    __shared__ bool join[2];
    __shared__ int kept, place[W];
    StepStream<D> st;
    st.init(plan_bytes(c.n_seqs), W, warp, a.depth);
    // A piece is a row of D + 2 floats for each row of the job: output, maximum, sum.  A warp's last piece
    // takes its ring, which has run dry by then; one of a job that ends inside the run takes one of the
    // CTA's few places behind the rings, or the workspace when they are gone.
    const int piece = min(a.tokens * a.group, R) * (D + 2);
    if (threadIdx.x == 0) kept = 0;
    auto piece_at = [&](int k) {
        const int i = k >> 1;
        if (k & 1) return reinterpret_cast<float*>(smem + plan_bytes(c.n_seqs) + i * a.depth * StepStream<D>::kSlot);
        if (place[i] < a.places) return reinterpret_cast<float*>(smem + a.first_off) + place[i] * piece;
        return a.first + (static_cast<size_t>(blockIdx.x) * W + i) * piece;
    };
    pdl_launch_dependents();
    pdl_wait();
    const Plan p = make_plan<32 * W>(c, a.jobs, gridDim.x * W, smem, blockIdx.x == 0 ? &g_kv_attend_error : nullptr);
    if (a.n_rt > 1 && blockIdx.x == 0)
        for (int b = threadIdx.x; b <= c.n_seqs; b += 32 * W) a.pre[b] = p.pre[b];
    const long long w = static_cast<long long>(blockIdx.x) * W + warp;
    const long long u0 = p.runs.start(w);
    const int n = static_cast<int>(p.runs.start(w + 1) - u0);
    if (lane < 2) pieces[2 * warp + lane].job = -1;
    __syncwarp();
    const int rows = a.tokens * a.group;
    if (n > 0) {
        QueryTile<D, NT> q;
        RowState<D, NT> rs;
        int b = 0, job = 0, len = 0, ub = 0, ul = 0, done = 0;
        bool gave_up = false;
        int left = 0;  // steps of the current sequence not yet begun, those of this run
        auto begin = [&](const StepAt& x) {
            b = x.b;
            len = x.len;
            ul = steps_of(len);
            job = x.job;
            ub = x.step;
            left = static_cast<int>(min(static_cast<long long>(p.pre[b + 1]) * p.jobs - (u0 + done), static_cast<long long>(n - done)));
        };
        {
            // the first queries are asked for before the whole GPU's first copies
            begin(st.start(a, p, u0, n));
            uint4 raw[NT][D / 32];
            q.request(a, b, job / a.n_rt, job % a.n_rt, raw);
            st.fill(a, p);
            if (a.n_rt == 1 && warp == 0 && lane < 2) {
                // while the copies travel: the jobs at the CTA's two ends, and who shares them
                const StepAt x = step_at(p, c.n_seqs, lane == 0 ? u0 : p.runs.start(w + W) - 1);
                cut[lane] = Piece{x.b, x.job, 0, 0};
                share[lane] = share_of<W>(p.pre, c.n_seqs, p.jobs, p.runs, x.b, x.job);
            }
            __syncwarp();
            q.arrange(a, job % a.n_rt, len, raw);
        }
        while (done < n && !gave_up) {
            if (left == 0) begin(step_at(p, c.n_seqs, u0 + done));
            // a job, or the part of it in this run
            const int first = ub, take = min(ul - ub, n - done);
            const int h = job / a.n_rt, rt = job - h * a.n_rt;
            if (done > 0) q.load(a, b, h, rt, len);
            rs.clear();
            for (int i = 0; i < take; ++i, ++ub) {
                if (!st.wait()) {
                    st.drain(done + i);
                    gave_up = true;
                    break;
                }
                const int j = ub * kStep;
                if (j < q.max_lim) {
                    uint32_t found = 3u;
                    if (st.absent) {
                        found = st.found();
                        if (j + kKvTokens >= len) found |= 2u;  // behind the last slot: not copied, and not missed
                    }
                    if ((ub & 7) == 7) rs.settle();
                    // the slot is refilled as soon as its V codes are in registers
                    if constexpr (NT == 1) {
                        uint32_t pf[2][NT][2], v[2][2][D / 32];
                        int2 index = make_int2(-1, -1);
                        if (kScores) index = st.unit_index();
                        rs.template weigh<2, 0, kScores>(q, st.unit(), j, len, found, a.scale2, pf, v, a.scores, a.pitch, index);
                        st.next(a, p);
                        rs.template output<2, 0>(pf, v);
                    } else {
                        uint32_t pf[1][NT][2], v[1][2][D / 32];
                        rs.template weigh<1, 0, false>(q, st.unit(), j, len, found & 1u, a.scale2, pf, v, nullptr, 0, make_int2(-1, -1));
                        rs.template output<1, 0>(pf, v);
                        const bool second = j + kKvTokens < q.max_lim;
                        if (second)
                            rs.template weigh<1, 1, false>(q, st.unit() + kv_unit_bytes(D), j + kKvTokens, len, found >> 1, a.scale2, pf, v,
                                                 nullptr, 0, make_int2(-1, -1));
                        st.next(a, p);
                        if (second) rs.template output<1, 1>(pf, v);
                    }
                } else {
                    st.next(a, p);
                }
            }
            if (gave_up) break;
            rs.settle();
            const bool whole = first == 0 && ub == ul;
            const int k = 2 * warp + (done + take == n ? 1 : 0);
            if (!whole && (k & 1) == 0) {
                if (lane == 0) place[warp] = atomicAdd(&kept, 1);
                __syncwarp();
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float v[D / 8];
                    const float sum = rs.finish(nt, e, v);
                    const int rl = nt * 8 + 2 * t + e, r = rt * R + rl;
                    if (r >= rows) continue;
                    if (whole) {
                        store_row(a, b, h, r, (D / 8) * g, v, rs.top(nt, e), sum);
                    } else {
                        float* dst = piece_at(k) + rl * (D + 2);
#pragma unroll
                        for (int i = 0; i < D / 8; i += 2)
                            *reinterpret_cast<float2*>(dst + (D / 8) * g + i) = make_float2(v[i], v[i + 1]);
                        if (g == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(rs.top(nt, e), sum);
                    }
                }
            if (!whole && lane == 0) pieces[k] = Piece{b, job, first, ub};
            done += take;
            left -= take;
            if (ub == ul) { ub = 0; ++job; }
        }
    }
    // rows of sequences without slots
    for (int b = blockIdx.x; b < c.n_seqs; b += gridDim.x) {
        if (p.len[b] != 0) continue;
        const int hq = c.heads * a.group;
        for (int i = threadIdx.x; i < a.tokens * hq * (D / 8); i += 32 * W) {
            const int x = i / (D / 8), tok = x / hq, head = x - tok * hq, col = 8 * (i % (D / 8));
            *reinterpret_cast<uint4*>(a.out + b * a.os[0] + tok * a.os[1] + head * a.os[2] + col) = make_uint4(0, 0, 0, 0);
            if (col == 0) store_lse(a, b, tok, head, 0.f, 0.f);
        }
    }
    __syncthreads();
    // Neighbouring pieces of one job meet here, in order, its rows dealt to the warps; a job that ends up
    // whole is finished, the others (at most the CTA's first and last) go to the workspace.
    Piece mine{0, -1, 0, 0};  // lane k: piece k
    if (lane < 2 * W) mine = pieces[lane];
    const uint32_t valid = __ballot_sync(0xffffffffu, mine.job >= 0);
    const uint32_t lower = valid & ((1u << lane) - 1u);
    const int prev = lower ? 31 - __clz(lower) : 0;
    const int my_h = a.n_rt == 1 ? mine.job : mine.job / a.n_rt, my_steps = mine.job >= 0 ? steps_of(p.len[mine.b]) : 0;
    const int pb = __shfl_sync(0xffffffffu, mine.b, prev), pj = __shfl_sync(0xffffffffu, mine.job, prev);
    const uint32_t heads = __ballot_sync(0xffffffffu, mine.job >= 0 && (!lower || pb != mine.b || pj != mine.job));
    // the groups of pieces of one job each: only the first and the last can be cut by the CTA's borders
    const int groups = __popc(heads), k_last = groups > 0 ? 31 - __clz(heads) : 0, k_first = groups > 0 ? __ffs(heads) - 1 : 0;
    auto members_of = [&](int k) {
        const uint32_t above = heads & ~((2u << k) - 1u);
        return valid & ~((1u << k) - 1u) & (above ? (above & (0u - above)) - 1u : 0xffffffffu);
    };
    auto is_cut = [&](int k) {
        return __shfl_sync(0xffffffffu, mine.first, k) != 0 ||
               __shfl_sync(0xffffffffu, mine.end, 31 - __clz(members_of(k))) != __shfl_sync(0xffffffffu, my_steps, k);
    };
    const bool cut_first = groups > 0 && is_cut(k_first), cut_last = groups > 1 && is_cut(k_last);
    const int cuts = cut_first + cut_last;
    // which of the CTA's two end jobs a cut group is: bit i of ends for cut i
    auto end_of = [&](int k) {
        return __shfl_sync(0xffffffffu, mine.b, k) != cut[0].b || __shfl_sync(0xffffffffu, mine.job, k) != cut[0].job;
    };
    const int ends = (cut_first && end_of(k_first) ? 1 : 0) | (cut_last && end_of(k_last) ? 1 << (cuts - 1) : 0);
    {
        constexpr int C = 8, L = D / C, P = 32 / L;  // columns of a lane, lanes of a row, rows of a turn
        const int turns = (min(rows, R) + P - 1) / P;
        for (int item = warp; item < groups * turns; item += W) {
            const int gi = item / turns, r0 = (item - gi * turns) * P;
            uint32_t hs = heads;
            for (int i = 0; i < gi; ++i) hs &= hs - 1;
            const int k = __ffs(hs) - 1;
            const uint32_t members = members_of(k);
            const int jb = __shfl_sync(0xffffffffu, mine.b, k), jj = __shfl_sync(0xffffffffu, mine.job, k);
            const int h = __shfl_sync(0xffffffffu, my_h, k), rt = jj - h * a.n_rt;
            const bool whole = !(gi == 0 ? cut_first : (gi == groups - 1 && cut_last));
            const int rl = r0 + lane / L, col = C * (lane % L);
            if (rl >= min(R, rows - rt * R)) continue;
            // the warps' last pieces with loads that do not wait for one another; first pieces are few
            float m = kNone, sum = 0.f, v[C], pm[W];
            const int ring0 = plan_bytes(c.n_seqs) + rl * (D + 2) * 4, ring_step = a.depth * StepStream<D>::kSlot;
            constexpr uint32_t kFirst = 0x55555555u;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                pm[i] = (members >> (2 * i + 1) & 1u) ? smem_at<float>(ring0 + i * ring_step + 4 * D) : kNone;
                m = fmaxf(m, pm[i]);
            }
            for (uint32_t x = members & kFirst; x; x &= x - 1) m = fmaxf(m, piece_at(__ffs(x) - 1)[rl * (D + 2) + D]);
#pragma unroll
            for (int y = 0; y < C; ++y) v[y] = 0.f;
            auto take = [&](float f, const float2 (&z)[C / 2], float l) {
                sum += l * f;
#pragma unroll
                for (int y = 0; y < C; y += 2) {
                    v[y] += z[y / 2].x * f;
                    v[y + 1] += z[y / 2].y * f;
                }
            };
            for (uint32_t x = members & kFirst; x; x &= x - 1) {
                const float* src = piece_at(__ffs(x) - 1) + rl * (D + 2);
                float2 z[C / 2];
#pragma unroll
                for (int y = 0; y < C / 2; ++y) z[y] = *reinterpret_cast<const float2*>(src + col + 2 * y);
                take(ex2(src[D] - m), z, src[D + 1]);
            }
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const bool on = members >> (2 * i + 1) & 1u;
                float2 z[C / 2];
#pragma unroll
                for (int y = 0; y < C / 2; ++y)
                    z[y] = on ? smem_at<float2>(ring0 + i * ring_step + 4 * (col + 2 * y)) : make_float2(0.f, 0.f);
                take(ex2(pm[i] - m), z, on ? smem_at<float>(ring0 + i * ring_step + 4 * D + 4) : 0.f);
            }
            if (whole) {
                store_row(a, jb, h, rt * R + rl, col, v, m, sum);
            } else {
                const size_t pi = (static_cast<size_t>(blockIdx.x) * 2 + (gi > 0 && cut_first ? 1 : 0)) * R + rl;
                float4* dst = reinterpret_cast<float4*>(a.part + pi * D + col);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                if (col == 0) *reinterpret_cast<float2*>(a.part_ml + pi * 2) = make_float2(m, sum);
            }
        }
    }
    if (cuts > 0 && a.n_rt == 1) {
        // one row tile: the last of a job's CTAs to arrive joins the partial sums, in CTA order
        __syncthreads();
        if (threadIdx.x < cuts) {
            const int i = ends >> threadIdx.x & 1;
            __threadfence();
            uint32_t* d = a.done + static_cast<size_t>(cut[i].b) * c.heads + cut[i].job;
            const bool last = atomicAdd(d, 1u) == static_cast<uint32_t>(share[i].n - 1);
            if (last) *d = 0;
            __threadfence();
            join[threadIdx.x] = last;
        }
        __syncthreads();
        for (int i = warp; i < cuts * rows; i += W) {
            const int x = i / rows, e = ends >> x & 1;
            if (join[x]) join_row<D, NT>(a, share[e], cut[e].b, cut[e].job, 0, i - x * rows);
        }
    }
    if (lane == 0 && n > 0 && st.absent) atomicOr(&g_kv_attend_error, kKvErrPage);
}

// ---------------------------------------------------------------------------
// Joins the partial sums of the jobs cut between CTAs when a KV head's rows fill
// several tiles (their jobs have no arrival counters).  One warp per row.  Bound
// by its chain of loads: 7 us by itself for 1280 rows of 64 columns.
// ---------------------------------------------------------------------------
constexpr int kCbWarps = 4;

template <int D, int NT>
__global__ void __launch_bounds__(32 * kCbWarps) kv_combine_kernel(const KvAttendArgs a, const int ctas) {
    const KvView& c = a.c;
    const int hq = c.heads * a.group;
    pdl_launch_dependents();
    pdl_wait();
    const long long item = static_cast<long long>(blockIdx.x) * kCbWarps + (threadIdx.x >> 5);
    if (item >= static_cast<long long>(c.n_seqs) * a.tokens * hq) return;
    const long long bt = item / hq;
    const int head = static_cast<int>(item - bt * hq), b = static_cast<int>(bt / a.tokens);
    const int tok = static_cast<int>(bt - static_cast<long long>(b) * a.tokens);
    const int h = head / a.group, r = tok * a.group + head - h * a.group, rt = r / (8 * NT);
    const Runs runs(a.pre[c.n_seqs], c.n_seqs, a.jobs, ctas * at_warps(NT));
    const Share s = share_of<at_warps(NT)>(a.pre, c.n_seqs, a.jobs, runs, b, h * a.n_rt + rt);
    if (s.n > 1) join_row<D, NT>(a, s, b, h, rt, r);  // else finished by its CTA, or empty
}

// ---------------------------------------------------------------------------
// Accumulated weight: mass_j += sum over the rows of exp2(score - lse), from the
// scores that the pass over the cache has kept: a lane a slot, 32 slots a step, a
// slot's sum in row order.  16 sequences of 2000 to 4100 slots, 8 heads of 8 rows:
// 14 us by itself, 43 with the attention.
// ---------------------------------------------------------------------------
constexpr int kSmWarps = 8;

template <int P>
__global__ void __launch_bounds__(32 * kSmWarps, 4) kv_score_mass_kernel(const KvAttendArgs a) {
    constexpr int B = P == 8 ? 2 : 4;  // steps at once; four of eight rows spill (36.6 against 36.4 us)
    extern __shared__ __align__(128) char smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const KvView& c = a.c;
    pdl_launch_dependents();
    pdl_wait();
    const Plan p = make_plan<32 * kSmWarps>(c, a.jobs, gridDim.x * kSmWarps, smem, nullptr);
    const long long w = static_cast<long long>(blockIdx.x) * kSmWarps + warp, u0 = p.runs.start(w);
    const int n = static_cast<int>(p.runs.start(w + 1) - u0);
    if (n == 0) return;
    const int rows = a.tokens * a.group;
    StepAt at = step_at(p, c.n_seqs, u0);
    float lse[P];
    for (int done = 0; done < n;) {
        const int ul = steps_of(at.len), take = min(ul - at.step, n - done);
        const bool none = a.counts && ld_l2(a.counts + at.b) <= 0;  // no query: no scores
#pragma unroll
        for (int r = 0; r < P; ++r) {
            lse[r] = INFINITY;  // padding rows and rows without keys weigh nothing
            if (r < rows) {
                const int tok = r / a.group, head = at.job * a.group + r - tok * a.group;
                const float x = ld_l2(a.lse2 + (static_cast<size_t>(at.b) * a.tokens + tok) * (c.heads * a.group) + head);
                if (x != -INFINITY) lse[r] = x;
            }
        }
        // several steps' loads at once: pages, then scores and sums
        for (int i0 = 0; i0 < take; i0 += B) {
            long long line[B];
            float s[B][P], was[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const int slot = (at.step + i0 + i) * kStep + lane;
                const bool on = i0 + i < take && slot < at.len && !none;
                const int page = on ? kv_page(c, at.b, slot) : -1;
                line[i] = page >= 0 ? static_cast<long long>(kv_line(c, page, at.job) + slot % c.page_size) : -1;
            }
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const float* src = a.scores + (line[i] >= 0 ? line[i] : 0) * P;
                const bool on = line[i] >= 0;
                if constexpr (P >= 4) {
#pragma unroll
                    for (int r = 0; r < P; r += 4) {
                        const uint4 x = on ? ld_l2_v4(src + r) : make_uint4(0, 0, 0, 0);
                        s[i][r] = __uint_as_float(x.x); s[i][r + 1] = __uint_as_float(x.y);
                        s[i][r + 2] = __uint_as_float(x.z); s[i][r + 3] = __uint_as_float(x.w);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < P; ++r) s[i][r] = on ? ld_l2(src + r) : 0.f;
                }
                was[i] = on ? ld_l2(c.mass + line[i]) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < B; ++i) {
                float add = 0.f;
#pragma unroll
                for (int r = 0; r < P; ++r)  // (a row whose lse is not a number gives nothing to the slots that it does not see)
                    if (r < rows && s[i][r] != -INFINITY) add += ex2(s[i][r] - lse[r]);
                if (line[i] >= 0) c.mass[line[i]] = was[i] + add;
            }
        }
        done += take;
        if (done < n) at = step_at(p, c.n_seqs, u0 + done);
    }
}

constexpr int kSmemPerSm = 226 * 1024;

// Ring slots per warp that fit next to the plan and `fixed` bytes when `ctas` CTAs share an SM, and the CTA's
// shared memory.
template <class Stream>
int ring_depth(int n_seqs, int warps, int ctas, int fixed, int* smem) {
    const int used = plan_bytes(n_seqs) + fixed, room = kSmemPerSm / ctas - 2048 - used;
    int depth = room / (warps * (Stream::kSlot + 16));
    depth = depth > 8 ? 8 : depth;
    *smem = used + Stream::bytes(warps, depth);
    return depth;
}

// Shared memory for pieces of jobs that end inside a run: two of eight rows, all of a CTA's with one row (where
// nearly every warp has one).  Room for eight of eight rows would take a slot of every ring.
constexpr int kKeptBytes = 8448;

template <int D, int NT>
dq_status_t attend(KvAttendArgs& a, cudaStream_t stream) {
    constexpr int W = at_warps(NT);
    DeviceInfo di;
    dq_status_t st = device_info(&di);
    if (st != DQ_OK) return st;
    int grid = di.sm_count * at_ctas(NT), smem = 0;
    if (grid * W > kAtMaxWarps) grid = kAtMaxWarps / W;
    const int rows = a.tokens * a.group, piece = (rows < 8 * NT ? rows : 8 * NT) * (D + 2) * 4;
    a.places = kKeptBytes / piece < W ? kKeptBytes / piece : W;
    a.depth = ring_depth<StepStream<D>>(a.c.n_seqs, W, at_ctas(NT), (a.places * piece + 127) / 128 * 128, &smem);
    a.first_off = smem - (a.places * piece + 127) / 128 * 128;
    // a piece fits in a ring of two slots
    static_assert(8 * NT * (D + 2) * 4 <= 2 * StepStream<D>::kSlot, "ring too small for a piece");
    if (a.depth < 2) return DQ_ERR_UNSUPPORTED;
    const auto kernel = NT == 1 && a.scores ? kv_attend_kernel<D, NT, NT == 1> : kv_attend_kernel<D, NT, false>;
    if ((st = allow_smem(kernel, smem)) != DQ_OK) return st;
    if ((st = launch_pdl(kernel, dim3(grid), 32 * W, smem, stream, 1, a)) != DQ_OK) return st;
    const long long items = static_cast<long long>(a.c.n_seqs) * a.tokens * a.c.heads * a.group;
    if (a.n_rt > 1)
        st = launch_pdl(kv_combine_kernel<D, NT>, dim3(static_cast<unsigned>((items + kCbWarps - 1) / kCbWarps)),
                    32 * kCbWarps, 0, stream, 1, a, grid);
    return st;
}

// The mass pass over kept scores of up to 8 rows.
dq_status_t score_mass(KvAttendArgs& a, cudaStream_t stream) {
    DeviceInfo di;
    const dq_status_t st = device_info(&di);
    if (st != DQ_OK) return st;
    a.jobs = Div(a.c.heads);
    const dim3 g(di.sm_count * 4);
    const int threads = 32 * kSmWarps, bytes = plan_bytes(a.c.n_seqs);
    switch (a.pitch) {
        case 1: return launch_pdl(kv_score_mass_kernel<1>, g, threads, bytes, stream, 1, a);
        case 2: return launch_pdl(kv_score_mass_kernel<2>, g, threads, bytes, stream, 1, a);
        case 4: return launch_pdl(kv_score_mass_kernel<4>, g, threads, bytes, stream, 1, a);
        default: return launch_pdl(kv_score_mass_kernel<8>, g, threads, bytes, stream, 1, a);
    }
}

// Query rows of a KV head from which the tensor-memory kernel of dq_kv_chunk.cu takes the call.  It costs about the
// same for 1 to 128 rows, this file's kernels cost more for every 16.  Here and there, in us, for 1 sequence of 8000
// slots and 32 KV heads, 4 of 2000 and 8, 16 of 4000 and 8: heads of 128 46, 29, 75 (32 rows), 58, 30, 102 (33) and
// 54, 22, 95; heads of 64 46, 23, 79 (64 rows), 54, 23, 95 (79) and 49, 20, 87.
constexpr int chunk_min(int head_dim) { return head_dim == 128 ? 33 : 65; }

// Row tiles of one warp: 8 rows when a KV head has no more, else 16.
int row_tiles(int rows) { return rows <= 8 ? 1 : 2; }

// What the mass pass may keep in the workspace: scores of up to 8 rows, or a line of sums for each of several tiles
// of 128.  Without that room it reads the keys a second time, a tile a launch.
constexpr size_t kMaxScores = size_t{1} << 30;

int score_pitch(int rows) { return rows <= 2 ? rows : (rows <= 4 ? 4 : 8); }

struct AttendWs {
    size_t part, ml, first, pre, lse2, scores, total;
};
AttendWs attend_ws(const dq_kv_cache_t& c, int tokens, int q_heads, bool mass) {
    const int nt = row_tiles(tokens * (q_heads / c.kv_heads));
    const bool chunk = tokens * (q_heads / c.kv_heads) >= chunk_min(c.head_dim);
    const size_t rows = chunk ? kv_chunk_part_rows() : static_cast<size_t>(kAtMaxWarps / at_warps(nt)) * 2 * 8 * nt;
    AttendWs w;
    w.part = 0;
    w.ml = align256(rows * c.head_dim * 4);
    w.first = w.ml + align256(rows * 8);
    w.pre = w.first + (chunk ? 0 : align256(static_cast<size_t>(kAtMaxWarps) * 8 * nt * (c.head_dim + 2) * 4));
    w.lse2 = w.pre + align256((static_cast<size_t>(c.n_seqs) + 1) * 4);
    w.scores = w.lse2 + (mass ? align256(static_cast<size_t>(c.n_seqs) * tokens * q_heads * 4) : 0);
    const int group_rows = tokens * (q_heads / c.kv_heads);
    const size_t line = static_cast<size_t>(c.n_pages) * c.kv_heads * c.page_size * sizeof(float);
    const size_t tiles = (group_rows + kChunkRows - 1) / kChunkRows;
    const size_t kept = line * (chunk ? (tiles > 1 ? tiles : 0) : score_pitch(group_rows));
    w.total = w.scores + (mass && (chunk || nt == 1) && group_rows > 0 && kept <= kMaxScores ? align256(kept) : 0);
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
    a.group = Div(r.q_heads / c.kv_heads);
    const float scale2 = r.scale * 1.44269504088896341f;
    a.scale2 = scale2 * kKey;
    a.done = c.arrivals + c.n_seqs;
    const AttendWs w = attend_ws(c, r.tokens, r.q_heads, r.accumulate != 0);
    char* base = static_cast<char*>(workspace);
    a.part = reinterpret_cast<float*>(base + w.part);
    a.part_ml = reinterpret_cast<float*>(base + w.ml);
    a.first = reinterpret_cast<float*>(base + w.first);
    a.pre = reinterpret_cast<int*>(base + w.pre);
    a.lse2 = r.accumulate ? reinterpret_cast<float*>(base + w.lse2) : nullptr;
    a.scores = w.total > w.scores ? reinterpret_cast<float*>(base + w.scores) : nullptr;
    const int rows = r.tokens * a.group, nt = row_tiles(rows);
    a.pitch = score_pitch(rows);
    KvAttendArgs whole = a;  // for dq_kv_chunk.cu, whose codes are whole numbers
    whole.scale2 = scale2;
    dq_status_t st;
    if (rows >= chunk_min(c.head_dim)) {
        st = launch_kv_chunk(whole, c.head_dim, stream);
    } else {
        a.n_rt = Div((rows + 8 * nt - 1) / (8 * nt));
        a.jobs = Div(c.kv_heads * a.n_rt);
        if (c.head_dim == 128) st = nt == 1 ? attend<128, 1>(a, stream) : attend<128, 2>(a, stream);
        else st = nt == 1 ? attend<64, 1>(a, stream) : attend<64, 2>(a, stream);
    }
    if (st != DQ_OK || !a.lse2) return st;
    return nt == 1 && a.scores ? score_mass(a, stream) : launch_kv_chunk_mass(whole, c.head_dim, whole.scores, stream);
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
