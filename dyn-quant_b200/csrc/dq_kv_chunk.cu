// dq_kv_chunk.cu -- attention over the paged 4-bit KV cache for many query rows
// per KV head (a prompt's chunk), on tcgen05 with the accumulators in tensor
// memory.  The same softmax and the same result as dq_kv_attend.cu's kernel.
//
// A tile is 128 query rows (token, query head) of one KV head, a block 128
// slots.  The (sequence, KV head, tile) jobs' blocks form one list cut into
// equal runs, one per CTA (one CTA an SM); pieces of jobs that a border cuts are
// joined by kv_chunk_combine_kernel.
//
// Roles of a CTA's fourteen warps, over the blocks i of its run:
//   loading (1)       page lookups and bulk copies of the block's units
//   dequantizing (4)  wait for the block's units (bulk copies), turn codes into
//                     f16 integers c - 8 in the MMA's shared-memory layout and
//                     the scales into FP32 constants.  K's tile is free again
//                     when S(i) is there, V's only after the block's softmax,
//                     so they are filled apart
//   MMA (1)           S(i) = Q K^T into one of two TMEM tiles, then, when the
//                     weights of i - 1 are there, O += P(i-1) V
//   softmax (8)       two threads per row, half of the block's slots (and of
//                     the output's columns) each: S(i) from TMEM, scores,
//                     weights, P(i) back to TMEM as the A operand; at a job's
//                     end O
// Everything hands over through mbarriers; every wait is bounded, and a CTA
// whose wait gave up sets the error word and leaves.
//
// K rows keep their words' column order (c0 c4 c1 c5 c2 c6 c3 c7): a word
// becomes one 16-byte chunk, and Q's columns are permuted alike.  V words hold
// two neighbouring slots of a column, which is a K-major pair of V^T as it is.
// Codes are exact in f16, scales and zeros are applied in FP32 around the
// products as in dq_kv_attend.cu; p' = p s_v w is rounded to f16.
//
// Measured: two sequences of 6000 and 8000 slots, 8 KV heads of 128 with 512 rows
// each, 31 GFLOP: 73 us, 0.42 PFLOP/s, and 9 us for the join.  A block takes 3900
// cycles, of which the exponentials are 1024, the MMAs 800; the softmax warps'
// other instructions and latencies bound it (45% of the issue slots are busy).
// Dequantizing and loading keep ahead of them.  Masks are applied after the loop
// over the scores, in the blocks that have one: inside it they cost 17 us.
#include "dq_kv_plan.cuh"

namespace dq {

namespace {

__device__ unsigned int g_kv_chunk_error;

constexpr int kBlk = 128;                  // slots of a block
constexpr int kUnits = kBlk / kKvTokens;   // units of a block
constexpr int kSoftWarps = 8, kSoft = 32 * kSoftWarps;  // two threads a row, half the columns each
constexpr int kMmaWarp = kSoftWarps + 4, kLoadWarp = kMmaWarp + 1;
constexpr int kCkThreads = 32 * (kLoadWarp + 1);
constexpr int kTile = kChunkRows;
constexpr int kChunkCtas = 160;            // bound on the grid (workspace sizing)

// Shared memory, offsets from a 1024-byte boundary.  Operand tiles are 128-byte rows (64 f16 of K) in groups of
// eight rows, the 16-byte chunks of row r xor-ed with r mod 8 (the 128-byte swizzle).
template <int D>
struct CkSmem {
    static constexpr int kQ = 0;                                 // [D/64][128 rows]
    static constexpr int kOp = D / 64 * kTile * 128;             // bytes of Q and of K
    static constexpr int kK = kQ + kOp;                          // 2 x [D/64][128 slots]
    static constexpr int kVBytes = kBlk / 64 * D * 128;
    static constexpr int kV = kK + 2 * kOp;                      // 2 x [2][D columns], 64 slots a row
    static constexpr int kRawBytes = kUnits * kv_unit_bytes(D);
    static constexpr int kRaw = kV + 2 * kVBytes;                // 2 x the units of a block
    static constexpr int kPar = kRaw + 2 * kRawBytes;            // 4 x [4][128]: - (z_k - 8), s_k, s_v, z_v - 8
    static constexpr int kMiscBytes = 48;
    static constexpr int kMisc = kPar + 4 * 4 * kBlk * 4;        // 4 x (4 x largest s_v, 4 x slots there, 4 x not finite)
    static constexpr int kGot = kMisc + 256;                     // 2 x found units
    static constexpr int kTop = kGot + 128;                      // 2 x [2 halves][128] largest score of a row's half
    static constexpr int kSums = kTop + 4 * kTile * 4;           // [2 halves][128] x 2: sum of weights, of zeros' share
    static constexpr int kQSum = kSums + 4 * kTile * 4;          // [2 halves][128] sums of q
    static constexpr int kBars = kQSum + 2 * kTile * 4;
    static constexpr int kTotal = kBars + 128;
};

// Barriers (8 bytes each).  Each but the last two is a pair, one for the even and one for the odd blocks.  S full also
// says that K has been read, V free that the block's product is in O, done that every product has ended.
enum { kRawFull = 0, kKFull = 2, kVFull = 4, kVFree = 6, kSFull = 8, kPFull = 10, kRawFree = 12, kQFull = 14, kDone = 15 };

// Tensor memory columns: two S tiles, O, two P tiles (f16 pairs).
constexpr uint32_t kTmS = 0, kTmO = 256, kTmP = 384, kTmCols = 512;

__device__ __forceinline__ void tm_alloc(uint32_t smem_dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tm_dealloc(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void tm_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Arrives on the barrier when the MMAs issued so far have completed.
__device__ __forceinline__ void tm_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// A K-major operand tile with the 128-byte swizzle: start address and the 1024 bytes between groups of eight rows in
// units of 16 bytes, descriptor version 1, swizzle mode 2.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// f16 x f16 -> f32, both operands K-major, M = 128, N = n.
__host__ __device__ constexpr uint32_t mma_shape(int n) {
    return (1u << 4) | (static_cast<uint32_t>(n / 8) << 17) | (static_cast<uint32_t>(kTile / 16) << 24);
}
__device__ __forceinline__ void tm_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"(add ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void tm_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(shape), "r"(add ? 1u : 0u)
        : "memory");
}

// 32 columns of the warp's 32 rows, one row a thread.
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// f16 pairs c - 8 of the nibbles at bits 0..3 / 16..19 and 4..7 / 20..23.
__device__ __forceinline__ uint32_t low_f16(uint32_t w) {
    return hsub2_u32(lop3_and_or(w, 0x000F000Fu, 0x64006400u), 0x64086408u);  // (1024 + c) - 1032
}
__device__ __forceinline__ uint32_t high_f16(uint32_t w) {
    return hsub2_u32(lop3_and_or(w, 0x00F000F0u, 0x54005400u), 0x54805480u);  // (64 + c) - 72
}

__device__ __forceinline__ void sts_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Walks the blocks of a CTA's run; every role keeps its own.
struct Walk {
    StepAt at;
    int blocks;  // of the job

    __device__ __forceinline__ void set(const Plan& p, int n_seqs, long long u) {
        at = step_at(p, n_seqs, u);
        blocks = steps_of<kBlk>(at.len);
    }
    // The next block; true when it begins another job.
    __device__ __forceinline__ bool next(const Plan& p, int n_seqs, long long u) {
        if (++at.step < blocks) return false;
        if (at.job + 1 < static_cast<int>(p.jobs)) {
            ++at.job;
            at.step = 0;
        } else {
            set(p, n_seqs, u);
        }
        return true;
    }
};

// Copies a block's units, the index of each in its lane (negative: none; `got` has the others' bits), one copy for
// units side by side in memory: a copy's issue takes some 80 cycles of the loading warp whatever its size.
template <int D>
__device__ __forceinline__ void copy_units(const KvView& c, uint32_t dst, int index, uint32_t got, int lane, uint32_t bar) {
    const int before = __shfl_up_sync(0xffffffffu, index, 1);
    const bool begins = index >= 0 && (lane == 0 || before + 1 != index || before < 0);
    const uint32_t ends = __ballot_sync(0xffffffffu, begins) | ~got;
    if (begins)
        bulk_g2s(dst + lane * kv_unit_bytes(D), c.units + static_cast<size_t>(index) * kv_unit_bytes(D),
                 __ffs(ends >> (lane + 1)) * kv_unit_bytes(D), bar);
}

// One unit's keys into the operand tile [D/64][128 slots]: a lane half a row, a word a chunk.
template <int D>
__device__ __forceinline__ void unpack_keys(const char* raw, char* tile, int u, int lane) {
    constexpr int N = D / 16;  // words of a lane
    const int row = lane & 15, half = lane >> 4;
    char* to = tile + (half * N / 8) * (kBlk * 128) + (u * kKvTokens + row) * 128;
#pragma unroll
    for (int i4 = 0; i4 < N / 4; ++i4) {
        const uint4 w4 = *reinterpret_cast<const uint4*>(raw + row * (D / 2) + half * (D / 4) + 16 * i4);
        const uint32_t ws[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w = ws[j], x = w >> 8;
            *reinterpret_cast<uint4*>(to + ((((half * N + 4 * i4 + j) % 8) ^ (row & 7)) << 4)) =
                make_uint4(low_f16(w), high_f16(w), low_f16(x), high_f16(x));
        }
    }
}

// Half of a query row's columns into the operand tile [D/64][128 rows], permuted as the keys' words are; their sum.
template <int D>
__device__ __forceinline__ float place_query(const uint16_t* src, bool on, char* tile, int row, int half) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const int ch = half * (D / 16) + i;
        const uint4 w = on ? ld_l2_v4(src + half * (D / 2) + 8 * i) : make_uint4(0, 0, 0, 0);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) s += h2f_bits(lo16(v[k])) + h2f_bits(hi16(v[k]));
        *reinterpret_cast<uint4*>(tile + ch / 8 * (kTile * 128) + row * 128 + (((ch % 8) ^ (row & 7)) << 4)) =
            make_uint4(__byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632), __byte_perm(w.y, w.w, 0x5410),
                       __byte_perm(w.y, w.w, 0x7632));
    }
    return s;
}

template <int D>
__global__ void __launch_bounds__(kCkThreads, 1) kv_chunk_kernel(const KvAttendArgs a) {
    using S = CkSmem<D>;
    extern __shared__ char dyn[];
    __shared__ uint32_t tm_base;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const KvView& c = a.c;
    const uint32_t smem0 = (smem_u32(dyn) + plan_bytes(c.n_seqs) + 1023u) & ~1023u;
    const uint32_t bars = smem0 + S::kBars;
    if (warp == kMmaWarp) tm_alloc(smem_u32(&tm_base), kTmCols);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars + 8 * (kRawFull + i), 1);
            mbar_init(bars + 8 * (kRawFree + i), 128);
            mbar_init(bars + 8 * (kKFull + i), 128);
            mbar_init(bars + 8 * (kVFull + i), 128);
            mbar_init(bars + 8 * (kVFree + i), 1);
            mbar_init(bars + 8 * (kSFull + i), 1);
            mbar_init(bars + 8 * (kPFull + i), kSoft);
        }
        mbar_init(bars + 8 * kQFull, kSoft);
        mbar_init(bars + 8 * kDone, 1);
        fence_mbar_init();
    }
    tm_before_sync();
    __syncthreads();
    tm_after_sync();
    const uint32_t tm = tm_base;
    pdl_launch_dependents();
    pdl_wait();
    const Plan p = make_plan<kCkThreads, kBlk>(c, a.jobs, gridDim.x, dyn, blockIdx.x == 0 ? &g_kv_chunk_error : nullptr);
    if (blockIdx.x == 0)
        for (int b = tid; b <= c.n_seqs; b += kCkThreads) a.pre[b] = p.pre[b];
    const long long u0 = p.runs.start(blockIdx.x);
    const int n = static_cast<int>(p.runs.start(blockIdx.x + 1) - u0);
    const int rows = a.tokens * a.group;
    // A warp whose wait gave up waits no more but takes every other step of its loop, so that nobody stays behind
    // at a barrier; the output is not valid then.
    bool dead = false;
    auto wait = [&](int bar, int parity) {
        if (dead) return;
        dead = !__all_sync(0xffffffffu, mbar_wait_bounded(bars + 8 * bar, parity & 1));
        if (dead && lane == 0) atomicOr(&g_kv_chunk_error, kKvErrWait);
    };
    // The MMA warp's end: tensor and shared memory are let go only when its products have ended, also after a wait that
    // gave up (a barrier of its own, since the others' phases may then lie behind).
    auto drain = [&](int bar) {
        if (lane == 0) tm_commit(bars + 8 * bar);
        __syncwarp();
        if (!mbar_wait_bounded(bars + 8 * bar, 0) && lane == 0) atomicOr(&g_kv_chunk_error, kKvErrWait);
    };
    Walk at;
    if (n > 0) at.set(p, c.n_seqs, u0);

    if (n > 0 && warp < kSoftWarps) {
        // ---- softmax
        constexpr int H = kBlk / 2;
        const int trow = 32 * (warp & 3) + lane, half = warp >> 2;
        const uint32_t lanes = tm + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        char* const base = dyn + (smem0 - smem_u32(dyn));
        auto word = [&](int off) -> float* { return reinterpret_cast<float*>(base + off); };
        float m = kNone, l = 0.f, zs = 0.f, vw = 0.f, qsum = 0.f;
        int lim = 0, r = 0, cuts = 0;
        bool begins = true;
        // the thread's half of the row's columns into the operand tile
        auto load_q = [&]() {
            const int h = at.at.job / a.n_rt, rt = at.at.job - h * a.n_rt;
            r = rt * kTile + trow;
            const int tok = r / a.group;
            const int cnt = a.counts ? min(max(ld_l2(a.counts + at.at.b), 0), a.tokens) : a.tokens;
            const bool on = r < rows && tok < cnt;
            lim = on ? min(max(at.at.len - cnt + tok + 1, 0), at.at.len) : 0;
            const uint16_t* src = a.q + at.at.b * a.qs[0] + tok * a.qs[1] + (h * a.group + r - tok * a.group) * a.qs[2];
            word(S::kQSum)[half * kTile + trow] = place_query<D>(src, on, base + S::kQ, trow, half);
            fence_async_smem();
            mbar_arrive(bars + 8 * kQFull);
            named_bar_sync(2, kSoft);
            qsum = word(S::kQSum)[trow] + word(S::kQSum)[kTile + trow];
        };
        load_q();
        int first = at.at.step;
        for (int i = 0; i < n; ++i) {
            const int buf = i & 1, step = at.at.step;
            wait(kSFull + buf, i >> 1);
            tm_after_sync();
            const float* par = word(S::kPar + (i & 3) * (4 * kBlk * 4)) + half * H;
            const float* misc = word(S::kMisc + (i & 3) * S::kMiscBytes);
            uint32_t va[32], vb[32];
            tm_ld32(lanes + kTmS + buf * kBlk + half * H, va);
            tm_ld32(lanes + kTmS + buf * kBlk + half * H + 32, vb);
            f2 s[H / 2];
            float top = -INFINITY;
            tm_wait_ld();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t (&v)[32] = k == 0 ? va : vb;
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 z = *reinterpret_cast<const float4*>(par + 32 * k + j);
                    const float4 sc = *reinterpret_cast<const float4*>(par + kBlk + 32 * k + j);
                    s[16 * k + j / 2] = fma2(f2(z.x, z.y), f2(qsum), f2(__uint_as_float(v[j]), __uint_as_float(v[j + 1]))) * f2(sc.x, sc.y);
                    s[16 * k + j / 2 + 1] =
                        fma2(f2(z.z, z.w), f2(qsum), f2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]))) * f2(sc.z, sc.w);
                }
            }
            const int left = lim - step * kBlk - half * H;  // slots of the half block that the row sees
            const uint2 there = *reinterpret_cast<const uint2*>(misc + 4 + 2 * half);
            if (left < H || (there.x & there.y) != 0xffffffffu) {
#pragma unroll
                for (int j = 0; j < H; j += 2) {
                    const uint32_t ok = (j < 32 ? there.x : there.y) >> (j & 31);
                    s[j / 2] = f2(j < left && (ok & 1u) ? s[j / 2].x() : -INFINITY, j + 1 < left && (ok & 2u) ? s[j / 2].y() : -INFINITY);
                }
            }
#pragma unroll
            for (int j = 0; j < H / 2; ++j) top = fmaxf(top, fmaxf(s[j].x(), s[j].y()));
            float* tops = word(S::kTop) + buf * 2 * kTile;
            tops[half * kTile + trow] = top;
            named_bar_sync(3 + (warp & 3), 64);  // the two warps of these rows
            top = fmaxf(top, tops[(half ^ 1) * kTile + trow]);
            // a new maximum or a larger V scale (the same for all rows)
            const float4 bg = *reinterpret_cast<const float4*>(misc);
            const float big = fmaxf(fmaxf(bg.x, bg.y), fmaxf(bg.z, bg.w));
            if (begins) {
                m = kNone;
                l = zs = 0.f;
                vw = 2147483648.0f;  // 2^31 brings the smallest FP16 scale, 2^-24, to 2^7
            }
            // value rows that are not finite (their scales and zeros are 0 here): the output of a row that sees one
            // is not either
            const uint2 odd = *reinterpret_cast<const uint2*>(misc + 8 + 2 * half);
            if ((odd.x | odd.y) != 0) {
                const unsigned long long sees = left >= H ? ~0ull : (1ull << max(left, 0)) - 1ull;
                if (((static_cast<unsigned long long>(odd.y) << 32 | odd.x) & sees) != 0) zs = NAN;
            }
            if (__any_sync(0xffffffffu, top > m + kLazy || big * vw > 128.f)) {
                float ratio = 1.f;
                if (big * vw > 128.f) {
                    // 2^(7 - e) with 2^(e-1) <= big < 2^e
                    const float nw = __uint_as_float((260u - (__float_as_uint(big) >> 23)) << 23);
                    ratio = __uint_as_float(__float_as_uint(nw) - __float_as_uint(vw) + 0x3F800000u);  // nw / vw, powers of two
                    vw = nw;
                }
                const float now = fmaxf(m, top), f = now == m ? 1.f : ex2(m - now), fr = f * ratio;
                m = now;
                l *= fr;
                zs *= fr;
                if (!begins) {
                    // O is the softmax warps' once the last block's product is in it
                    wait(kVFree + (buf ^ 1), (i - 1) >> 1);
                    tm_after_sync();
#pragma unroll 1
                    for (int k = 0; k < D / 64; ++k) {
                        uint32_t v[32];
                        const uint32_t o = lanes + kTmO + half * (D / 2) + 32 * k;
                        tm_ld32(o, v);
                        tm_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * fr);
                        tm_st32(o, v);
                    }
                    tm_wait_st();
                }
            }
            // 2^(s - m) w at once: l too is in units of 1 / w
            const f2 shift(static_cast<float>(static_cast<int>(__float_as_uint(vw) >> 23) - 127) - m);
            f2 l2(0.f), z2(0.f);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t pk[16];
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 w4 = *reinterpret_cast<const float4*>(par + 2 * kBlk + 32 * k + j);
                    const float4 z4 = *reinterpret_cast<const float4*>(par + 3 * kBlk + 32 * k + j);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const f2 d = s[16 * k + j / 2 + e] + shift, x(ex2(d.x()), ex2(d.y()));
                        const f2 pr = x * f2(e ? w4.z : w4.x, e ? w4.w : w4.y);
                        l2 = l2 + x;
                        z2 = fma2(pr, f2(e ? z4.z : z4.x, e ? z4.w : z4.y), z2);
                        pk[j / 2 + e] = pack_f32(pr.x(), pr.y());
                    }
                }
                tm_st16(lanes + kTmP + buf * 64 + half * 32 + 16 * k, pk);
            }
            l += l2.x() + l2.y();
            zs += z2.x() + z2.y();
            tm_wait_st();
            tm_before_sync();
            mbar_arrive(bars + 8 * (kPFull + buf));
            begins = false;
            // the job's end, or the run's
            const StepAt was = at.at;
            const int blocks = at.blocks, row = r;
            const bool last = i + 1 == n, turn = last || at.next(p, c.n_seqs, u0 + i + 1);
            if (!turn) continue;
            float* sums = word(S::kSums);
            sums[half * kTile + trow] = l;
            sums[(2 + half) * kTile + trow] = zs;
            if (!last) load_q();  // S of the old rows is done; the new ones' can start
            else named_bar_sync(2, kSoft);
            const float inv_w = __uint_as_float(0x7F000000u - __float_as_uint(vw));
            const float lsum = (sums[trow] + sums[kTile + trow]) * inv_w, zsum = sums[2 * kTile + trow] + sums[3 * kTile + trow];
            wait(kVFree + buf, i >> 1);
            tm_after_sync();
            const bool whole = first == 0 && was.step + 1 == blocks;
            const int h = was.job / a.n_rt;
            const size_t pi = (static_cast<size_t>(blockIdx.x) * 2 + cuts) * kTile + trow;
#pragma unroll 1
            for (int k = 0; k < D / 64; ++k) {
                uint32_t v[32];
                const int col = half * (D / 2) + 32 * k;
                tm_ld32(lanes + kTmO + col, v);
                tm_wait_ld();
                if (row < rows) {
                    float o[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = (__uint_as_float(v[j]) - zsum) * inv_w;
                    if (whole) {
                        store_row(a, was.b, h, row, col, o, m, lsum);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<float4*>(a.part + pi * D + col + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                        if (col == 0) *reinterpret_cast<float2*>(a.part_ml + pi * 2) = make_float2(m, lsum);
                    }
                }
            }
            tm_before_sync();
            if (!whole) ++cuts;
            first = at.at.step;
            begins = true;
        }
    } else if (n > 0 && warp < kMmaWarp) {
        // ---- dequantizing
        const int dw = warp - kSoftWarps;
        char* const base = dyn + (smem0 - smem_u32(dyn));
        for (int i = 0; i < n; ++i) {
            const int buf = i & 1;
            wait(kRawFull + buf, i >> 1);
            if (i >= 2) wait(kSFull + buf, (i - 2) >> 1);
            const uint32_t got = lds_u32(smem0 + S::kGot + buf * 4);
            const char* raws = base + S::kRaw + buf * S::kRawBytes;
#pragma unroll 1
            for (int e = 0; e < 2; ++e) unpack_keys<D>(raws + (2 * dw + e) * kv_unit_bytes(D), base + S::kK + buf * S::kOp, 2 * dw + e, lane);
            {
                // scales and zeros, a lane a slot
                const int u = 2 * dw + (lane >> 4), slot = 32 * dw + lane;
                const bool on = (got >> u & 1u) && at.at.step * kBlk + slot < at.at.len;
                const uint2 pw = lds_v2(smem0 + S::kRaw + buf * S::kRawBytes + u * kv_unit_bytes(D) + kv_param_offset(D) + 8 * (lane & 15));
                float sv = on ? h2f_bits(lo16(pw.y)) : 0.f, zv = on ? h2f_bits(hi16(pw.y)) - 8.f : 0.f;
                const bool finite = fabsf(sv) + fabsf(zv) < INFINITY;
                if (!finite) sv = zv = 0.f;
                const uint32_t par = smem0 + S::kPar + (i & 3) * (4 * kBlk * 4) + 4 * slot, misc = smem0 + S::kMisc + (i & 3) * S::kMiscBytes;
                sts_u32(par, __float_as_uint(on ? 8.f - h2f_bits(hi16(pw.x)) : 0.f));
                sts_u32(par + 4 * kBlk, __float_as_uint(on ? h2f_bits(lo16(pw.x)) * a.scale2 : 0.f));
                sts_u32(par + 8 * kBlk, __float_as_uint(sv));
                sts_u32(par + 12 * kBlk, __float_as_uint(zv));
                float big = sv;
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                const uint32_t there = __ballot_sync(0xffffffffu, on), odd = __ballot_sync(0xffffffffu, !finite);
                if (lane == 0) {
                    sts_u32(misc + 4 * dw, __float_as_uint(big));
                    sts_u32(misc + 16 + 4 * dw, there);
                    sts_u32(misc + 32 + 4 * dw, odd);
                }
            }
            fence_async_smem();
            mbar_arrive(bars + 8 * (kKFull + buf));
            if (i >= 2) wait(kVFree + buf, (i - 2) >> 1);
            // V: a lane four column quads of a slot pair at a time; which quad (g1) and which two columns (g2)
            // come first differs among the lanes of a pair, so that the 32 words of a store lie in 32 banks.
            const int pr = lane >> 2, g = lane & 3, g1 = g & 1, g2 = g & 2;
#pragma unroll 1
            for (int e = 0; e < 2; ++e) {
                const int u = 2 * dw + e;
                const char* raw = raws + u * kv_unit_bytes(D);
                const int key = u * kKvTokens + 2 * pr, byte = 2 * (key % 64);  // the pair's first slot
                char* vt = base + S::kV + buf * S::kVBytes + key / 64 * (D * 128) + 512 * 4 * g;
                char* even[4];  // columns of quads g1, 2 + g1: in the order of their stores
                char* odd[4];   // of quads 1 - g1, 3 - g1
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int col = j ^ g2;
                    even[j] = vt + 512 * g1 + 128 * col + (byte ^ ((4 * g1 + col) << 4));
                    odd[j] = vt + 512 * (g1 ^ 1) + 128 * col + (byte ^ ((4 * (g1 ^ 1) + col) << 4));
                }
#pragma unroll
                for (int i4 = 0; i4 < D / 64; ++i4) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(raw + kv_v_offset(D) + pr * D + 64 * i4 + 16 * g);
                    const uint32_t ws[4] = {g1 ? w4.y : w4.x, g1 ? w4.x : w4.y, g1 ? w4.w : w4.z, g1 ? w4.z : w4.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t w = ws[k] >> (g2 * 4), x = ws[k] >> (8 - g2 * 4);
                        char* const* to = k & 1 ? odd : even;
                        const int at4 = 512 * 16 * i4 + 1024 * (k >> 1);
                        *reinterpret_cast<uint32_t*>(to[0] + at4) = low_f16(w);
                        *reinterpret_cast<uint32_t*>(to[1] + at4) = high_f16(w);
                        *reinterpret_cast<uint32_t*>(to[2] + at4) = low_f16(x);
                        *reinterpret_cast<uint32_t*>(to[3] + at4) = high_f16(x);
                    }
                }
            }
            fence_async_smem();
            mbar_arrive(bars + 8 * (kVFull + buf));
            mbar_arrive(bars + 8 * (kRawFree + buf));
            if (i + 1 < n) at.next(p, c.n_seqs, u0 + i + 1);
        }
    } else if (n > 0 && warp == kMmaWarp) {
        // ---- MMA
        int jobs = 0;
        bool begins = true, begins_before = true;
        auto output = [&](int i, bool start) {
            const int buf = i & 1;
            wait(kPFull + buf, i >> 1);
            wait(kVFull + buf, i >> 1);
            tm_after_sync();
            if (lane == 0) {
                const uint32_t vb = smem0 + S::kV + buf * S::kVBytes;
#pragma unroll
                for (int k = 0; k < kBlk / 16; ++k)
                    tm_mma_ts(tm + kTmO, tm + kTmP + buf * 64 + 8 * k, operand(vb + k / 4 * (D * 128) + 32 * (k % 4)), mma_shape(D),
                              !(start && k == 0));
                tm_commit(bars + 8 * (kVFree + buf));
            }
            __syncwarp();
        };
        for (int i = 0; i < n; ++i) {
            const int buf = i & 1;
            if (begins) wait(kQFull, jobs);
            wait(kKFull + buf, i >> 1);
            tm_after_sync();
            if (lane == 0) {
                const uint32_t kb = smem0 + S::kK + buf * S::kOp;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    tm_mma_ss(tm + kTmS + buf * kBlk, operand(smem0 + S::kQ + k / 4 * (kTile * 128) + 32 * (k % 4)),
                              operand(kb + k / 4 * (kBlk * 128) + 32 * (k % 4)), mma_shape(kBlk), k > 0);
                tm_commit(bars + 8 * (kSFull + buf));
            }
            __syncwarp();
            if (i > 0) output(i - 1, begins_before);
            begins_before = begins;
            if (begins) ++jobs;
            begins = i + 1 < n && at.next(p, c.n_seqs, u0 + i + 1);
        }
        output(n - 1, begins_before);
        drain(kDone);
    } else if (n > 0) {
        // ---- loading: a lane a unit, a copy a run of units of one page
        bool absent = false;
        int asked = 0;
        for (int i = 0; i < n; ++i) {
            const int buf = i & 1, slot = at.at.step * kBlk + lane * kKvTokens;
            int index = -1;
            if (lane < kUnits && slot < at.at.len) {
                const int page = kv_page(c, at.at.b, slot);
                if (page >= 0) index = static_cast<int>((kv_line(c, page, at.at.job / a.n_rt) + slot % c.page_size) / kKvTokens);
                else absent = true;
            }
            if (i >= 2) {
                wait(kRawFree + buf, (i - 2) >> 1);
                wait(kRawFull + buf, (i - 2) >> 1);  // long ago, unless its readers gave up
            }
            if (dead) break;
            asked = i + 1;
            const uint32_t got = __ballot_sync(0xffffffffu, index >= 0), bar = bars + 8 * (kRawFull + buf);
            if (lane == 0) {
                sts_u32(smem0 + S::kGot + buf * 4, got);
                if (got) mbar_arrive_expect_tx(bar, __popc(got) * kv_unit_bytes(D));
                else mbar_arrive(bar);
            }
            __syncwarp();
            copy_units<D>(c, smem0 + S::kRaw + buf * S::kRawBytes, index, got, lane, bar);
            if (i + 1 < n) at.next(p, c.n_seqs, u0 + i + 1);
        }
        // the copies must end before the shared memory goes, whatever their readers have done
        for (int j = max(asked - 2, 0); j < asked; ++j) mbar_wait_bounded(bars + 8 * (kRawFull + (j & 1)), (j >> 1) & 1);
        if (absent) atomicOr(&g_kv_chunk_error, kKvErrPage);
    }
    // rows of sequences without slots
    for (int b = blockIdx.x; b < c.n_seqs; b += gridDim.x) {
        if (p.len[b] != 0) continue;
        const int hq = c.heads * a.group;
        for (int i = tid; i < a.tokens * hq * (D / 8); i += kCkThreads) {
            const int x = i / (D / 8), tok = x / hq, head = x - tok * hq, col = 8 * (i % (D / 8));
            *reinterpret_cast<uint4*>(a.out + b * a.os[0] + tok * a.os[1] + head * a.os[2] + col) = make_uint4(0, 0, 0, 0);
            if (col == 0) store_lse(a, b, tok, head, 0.f, 0.f);
        }
    }
    tm_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        tm_after_sync();
        tm_dealloc(tm, kTmCols);
    }
}

// Joins the partial sums of the jobs cut between CTAs: one warp per row.
constexpr int kCcWarps = 4;

template <int D>
__global__ void __launch_bounds__(32 * kCcWarps) kv_chunk_combine_kernel(const KvAttendArgs a, const int ctas) {
    const KvView& c = a.c;
    const int hq = c.heads * a.group;
    pdl_launch_dependents();
    pdl_wait();
    const long long item = static_cast<long long>(blockIdx.x) * kCcWarps + (threadIdx.x >> 5);
    if (item >= static_cast<long long>(c.n_seqs) * a.tokens * hq) return;
    const long long bt = item / hq;
    const int head = static_cast<int>(item - bt * hq), b = static_cast<int>(bt / a.tokens);
    const int tok = static_cast<int>(bt - static_cast<long long>(b) * a.tokens);
    const int h = head / a.group, r = tok * a.group + head - h * a.group, rt = r / kTile;
    const Runs runs(a.pre[c.n_seqs], c.n_seqs, a.jobs, ctas);
    const Share s = share_of<1>(a.pre, c.n_seqs, a.jobs, runs, b, h * a.n_rt + rt);
    if (s.n > 1) join_row<D, kTile / 8, 4>(a, s, b, h, rt, r);  // else finished by its CTA, or empty
}

// ---------------------------------------------------------------------------
// Accumulated weight: mass_j += sum over the rows of exp2(score - lse), from the
// keys once more now that every row's lse is known (the scores of up to 8 rows
// are kept by the pass over the cache instead, see dq_kv_attend.cu).  S^T = K Q^T
// has a slot a TMEM lane, so a thread adds its slot's weights over the tile's rows
// by itself, with the rows' sums of q and lse from shared memory.  One row tile's
// sums are added to mass at once; those of several go to lines of their own in the
// workspace, which kv_tile_mass_kernel (7 us by itself) adds to mass in tile order,
// or, where the lines would be too many, to mass by a launch a tile.  The two halves of
// the softmax warps take the blocks in turn, a slot's 128 rows a thread, and four S
// tiles keep the MMAs ahead of them: 41 us for the case above where one block at a
// time, its rows split over two threads, took 55.
// ---------------------------------------------------------------------------
template <int D>
struct CmSmem {
    static constexpr int kOp = D / 64 * kTile * 128;
    static constexpr int kQ = 0;
    static constexpr int kK = kOp;                               // 2 x
    static constexpr int kRawBytes = kUnits * kv_unit_bytes(D);
    static constexpr int kRaw = kK + 2 * kOp;                    // 4 x the units of a block
    static constexpr int kPar = kRaw + 4 * kRawBytes;            // 8 x [2][128]: - (z_k - 8), s_k
    static constexpr int kRow = kPar + 16 * kBlk * 4;            // [4][128]: sum of q (two halves), - lse, keys seen
    static constexpr int kIndex = kRow + 4 * kTile * 4;          // 16 x the block's units
    static constexpr int kThere = kIndex + 16 * kUnits * 4;      // 8 x (4 x slots there)
    static constexpr int kMisc = kThere + 8 * 16;                // 4 x found units; 4 x keys seen
    static constexpr int kBars = kMisc + 128;
    static constexpr int kTotal = kBars + 256;
};

// Barriers: four for the units' buffers and for the S tiles, two for K's tiles.  S full also says that K has been read,
// and a block's constants are kept until its S is free: the warps that fill them are at most six blocks ahead of those
// that read them, the loading warp ten.
enum { kCmRawFull = 0, kCmRawFree = 4, kCmSFull = 8, kCmSFree = 12, kCmKFull = 16, kCmQFull = 18, kCmDone = 19 };

template <int D>
__global__ void __launch_bounds__(kCkThreads, 1) kv_chunk_mass_kernel(const KvAttendArgs a, float* sums, const long long lines,
                                                                      const int rt0) {
    using S = CmSmem<D>;
    extern __shared__ char dyn[];
    __shared__ uint32_t tm_base;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const KvView& c = a.c;
    const uint32_t smem0 = (smem_u32(dyn) + plan_bytes(c.n_seqs) + 1023u) & ~1023u;
    const uint32_t bars = smem0 + S::kBars;
    char* const base = dyn + (smem0 - smem_u32(dyn));
    auto word = [&](int off) -> float* { return reinterpret_cast<float*>(base + off); };
    if (warp == kMmaWarp) tm_alloc(smem_u32(&tm_base), kTmCols);
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(bars + 8 * (kCmRawFull + i), 1);
            mbar_init(bars + 8 * (kCmRawFree + i), 128);
            mbar_init(bars + 8 * (kCmSFull + i), 1);
            mbar_init(bars + 8 * (kCmSFree + i), kTile);  // S and the block's constants have been read
        }
        for (int i = 0; i < 2; ++i) mbar_init(bars + 8 * (kCmKFull + i), 128);
        mbar_init(bars + 8 * kCmQFull, kSoft);
        mbar_init(bars + 8 * kCmDone, 1);
        fence_mbar_init();
    }
    tm_before_sync();
    __syncthreads();
    tm_after_sync();
    const uint32_t tm = tm_base;
    pdl_launch_dependents();
    pdl_wait();
    const Plan p = make_plan<kCkThreads, kBlk>(c, a.jobs, gridDim.x, dyn, nullptr);
    const long long u0 = p.runs.start(blockIdx.x);
    const int n = static_cast<int>(p.runs.start(blockIdx.x + 1) - u0);
    const int rows = a.tokens * a.group;
    bool dead = false;
    auto wait = [&](int bar, int parity) {
        if (dead) return;
        dead = !__all_sync(0xffffffffu, mbar_wait_bounded(bars + 8 * bar, parity & 1));
        if (dead && lane == 0) atomicOr(&g_kv_chunk_error, kKvErrWait);
    };
    // The MMA warp's end: tensor and shared memory are let go only when its products have ended, also after a wait that
    // gave up (a barrier of its own, since the others' phases may then lie behind).
    auto drain = [&](int bar) {
        if (lane == 0) tm_commit(bars + 8 * bar);
        __syncwarp();
        if (!mbar_wait_bounded(bars + 8 * bar, 0) && lane == 0) atomicOr(&g_kv_chunk_error, kKvErrWait);
    };
    Walk at;
    if (n > 0) at.set(p, c.n_seqs, u0);
    // Columns of S that have rows of the tile, by 32: the others are neither multiplied nor read (12 rows of 32 heads,
    // 3 sequences of 8476 to 16953 slots: 181 us with the attention, 207 with all; full tiles lose 1%).
    auto columns = [&]() {
        const int left = rows - (rt0 + at.at.job - at.at.job / a.n_rt * a.n_rt) * kTile;
        return min((left + 31) / 32 * 32, kTile);
    };

    if (n > 0 && warp < kSoftWarps) {
        const int trow = 32 * (warp & 3) + lane, half = warp >> 2;
        const uint32_t lanes = tm + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        int least = 0, cols = 0;  // keys that every row of the tile sees; the tile's columns
        auto load_q = [&]() {
            const int h = at.at.job / a.n_rt, rt = at.at.job - h * a.n_rt;
            const int r = (rt0 + rt) * kTile + trow, tok = r / a.group;
            const int cnt = a.counts ? min(max(ld_l2(a.counts + at.at.b), 0), a.tokens) : a.tokens;
            const bool on = r < rows && tok < cnt;
            const int head = h * a.group + r - tok * a.group;
            const uint16_t* src = a.q + at.at.b * a.qs[0] + tok * a.qs[1] + head * a.qs[2];
            word(S::kRow)[half * kTile + trow] = place_query<D>(src, on, base + S::kQ, trow, half);
            if (half == 0) {
                // rows that are padding or see no key weigh nothing
                float nl = -INFINITY;
                int lim = 0;
                if (on) {
                    const float x = ld_l2(a.lse2 + (static_cast<size_t>(at.at.b) * a.tokens + tok) * (c.heads * a.group) + head);
                    lim = min(max(at.at.len - cnt + tok + 1, 0), at.at.len);
                    if (x != -INFINITY) nl = -x;
                }
                word(S::kRow)[2 * kTile + trow] = nl;
                // (padding sees all, so that it costs no masks, but nothing where the sequence has no query at all:
                // 0 times a key that is not finite is not 0)
                reinterpret_cast<int*>(word(S::kRow))[3 * kTile + trow] = on ? lim : (cnt > 0 ? at.at.len : 0);
            }
            fence_async_smem();
            mbar_arrive(bars + 8 * kCmQFull);
            named_bar_sync(2, kSoft);
            if (half == 0) word(S::kRow)[trow] += word(S::kRow)[kTile + trow];
            int lim = reinterpret_cast<const int*>(word(S::kRow))[3 * kTile + trow];
            lim = __reduce_min_sync(0xffffffffu, lim);
            if (half == 0 && lane == 0) reinterpret_cast<int*>(word(S::kMisc))[4 + (warp & 3)] = lim;
            named_bar_sync(2, kSoft);
            const int4 l4 = *reinterpret_cast<const int4*>(word(S::kMisc) + 4);
            least = min(min(l4.x, l4.y), min(l4.z, l4.w));
            cols = columns();
        };
        load_q();
        for (int i = 0; i < n; ++i) {
            if ((i & 1) == half) {
                const int buf = i & 3, slot = at.at.step * kBlk + trow;
                wait(kCmSFull + buf, i >> 2);
                tm_after_sync();
                const float* par = word(S::kPar + (i & 7) * (2 * kBlk * 4));
                const float nz = par[trow], sk = par[kBlk + trow];
                const bool there = reinterpret_cast<const uint32_t*>(word(S::kThere + (i & 7) * 16))[warp & 3] >> lane & 1u;
                const int unit = reinterpret_cast<const int*>(word(S::kIndex + (i & 15) * (kUnits * 4)))[trow / kKvTokens];
                const bool all = (at.at.step + 1) * kBlk <= least;
                f2 add(0.f);
                auto weigh = [&](const float* row, const uint32_t (&x)[32]) {
                    f2 s[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 qs = *reinterpret_cast<const float4*>(row + j);
                        const float4 nl = *reinterpret_cast<const float4*>(row + 2 * kTile + j);
                        s[j / 2] = fma2(fma2(f2(nz), f2(qs.x, qs.y), f2(__uint_as_float(x[j]), __uint_as_float(x[j + 1]))), f2(sk), f2(nl.x, nl.y));
                        s[j / 2 + 1] =
                            fma2(fma2(f2(nz), f2(qs.z, qs.w), f2(__uint_as_float(x[j + 2]), __uint_as_float(x[j + 3]))), f2(sk), f2(nl.z, nl.w));
                    }
                    if (!all) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const int4 lim = *reinterpret_cast<const int4*>(row + 3 * kTile + j);
                            s[j / 2] = f2(slot < lim.x ? s[j / 2].x() : -INFINITY, slot < lim.y ? s[j / 2].y() : -INFINITY);
                            s[j / 2 + 1] = f2(slot < lim.z ? s[j / 2 + 1].x() : -INFINITY, slot < lim.w ? s[j / 2 + 1].y() : -INFINITY);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) add = add + f2(ex2(s[j].x()), ex2(s[j].y()));
                };
                if (cols == kTile) {
                    uint32_t v[2][32];
                    tm_ld32(lanes + buf * kTile, v[0]);
#pragma unroll
                    for (int k = 0; k < kTile / 32; ++k) {
                        tm_wait_ld();
                        if (k + 1 < kTile / 32) tm_ld32(lanes + buf * kTile + 32 * (k + 1), v[(k + 1) & 1]);
                        weigh(word(S::kRow) + 32 * k, v[k & 1]);
                    }
                } else {
#pragma unroll 1
                    for (int k = 0; k < cols; k += 32) {
                        uint32_t v[32];
                        tm_ld32(lanes + buf * kTile + k, v);
                        tm_wait_ld();
                        weigh(word(S::kRow) + k, v);
                    }
                }
                tm_before_sync();
                mbar_arrive(bars + 8 * (kCmSFree + buf));
                if (there) {
                    const long long line = static_cast<long long>(unit) * kKvTokens + trow % kKvTokens;
                    const float sum = add.x() + add.y();
                    if (a.n_rt == 1) atomicAdd(c.mass + line, sum);  // the slot's only one: no order, and nothing waits for it
                    else sums[(at.at.job - at.at.job / a.n_rt * a.n_rt) * lines + line] = sum;
                }
            }
            if (i + 1 < n && at.next(p, c.n_seqs, u0 + i + 1)) {
                named_bar_sync(2, kSoft);  // all have read the old rows' constants; S of them is done
                load_q();
            }
        }
    } else if (n > 0 && warp < kMmaWarp) {
        const int dw = warp - kSoftWarps;
        for (int i = 0; i < n; ++i) {
            const int buf = i & 1, from = i & 3;
            wait(kCmRawFull + from, i >> 2);
            if (i >= 2) wait(kCmSFull + ((i - 2) & 3), (i - 2) >> 2);
            const uint32_t got = reinterpret_cast<const uint32_t*>(word(S::kMisc))[from];
            const char* raw = base + S::kRaw + from * S::kRawBytes;
#pragma unroll 1
            for (int e = 0; e < 2; ++e) unpack_keys<D>(raw + (2 * dw + e) * kv_unit_bytes(D), base + S::kK + buf * S::kOp, 2 * dw + e, lane);
            const int u = 2 * dw + (lane >> 4), slot = 32 * dw + lane;
            const bool on = (got >> u & 1u) && at.at.step * kBlk + slot < at.at.len;
            const uint32_t pw = *reinterpret_cast<const uint32_t*>(raw + u * kv_unit_bytes(D) + kv_param_offset(D) + 8 * (lane & 15));
            float* par = word(S::kPar + (i & 7) * (2 * kBlk * 4));
            par[slot] = on ? 8.f - h2f_bits(hi16(pw)) : 0.f;
            par[kBlk + slot] = on ? h2f_bits(lo16(pw)) * a.scale2 : 0.f;
            const uint32_t there = __ballot_sync(0xffffffffu, on);
            if (lane == 0) reinterpret_cast<uint32_t*>(word(S::kThere + (i & 7) * 16))[dw] = there;
            fence_async_smem();
            mbar_arrive(bars + 8 * (kCmKFull + buf));
            mbar_arrive(bars + 8 * (kCmRawFree + from));
            if (i + 1 < n) at.next(p, c.n_seqs, u0 + i + 1);
        }
    } else if (n > 0 && warp == kMmaWarp) {
        int jobs = 0;
        uint32_t shape = 0;
        bool begins = true;
        for (int i = 0; i < n; ++i) {
            const int buf = i & 1;
            if (begins) {
                wait(kCmQFull, jobs++);
                shape = mma_shape(columns());
            }
            wait(kCmKFull + buf, i >> 1);
            if (i >= 4) wait(kCmSFree + (i & 3), (i - 4) >> 2);
            tm_after_sync();
            if (lane == 0) {
                const uint32_t kb = smem0 + S::kK + buf * S::kOp;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    tm_mma_ss(tm + (i & 3) * kTile, operand(kb + k / 4 * (kBlk * 128) + 32 * (k % 4)),
                              operand(smem0 + S::kQ + k / 4 * (kTile * 128) + 32 * (k % 4)), shape, k > 0);
                tm_commit(bars + 8 * (kCmSFull + (i & 3)));
            }
            __syncwarp();
            begins = i + 1 < n && at.next(p, c.n_seqs, u0 + i + 1);
        }
        drain(kCmDone);
    } else if (n > 0) {
        // ---- loading, as above
        int asked = 0;
        for (int i = 0; i < n; ++i) {
            const int buf = i & 3, slot = at.at.step * kBlk + lane * kKvTokens;
            int index = -1;
            if (lane < kUnits && slot < at.at.len) {
                const int page = kv_page(c, at.at.b, slot);
                if (page >= 0) index = static_cast<int>((kv_line(c, page, at.at.job / a.n_rt) + slot % c.page_size) / kKvTokens);
            }
            if (i >= 4) {
                wait(kCmRawFree + buf, (i - 4) >> 2);
                wait(kCmRawFull + buf, (i - 4) >> 2);
            }
            if (dead) break;
            asked = i + 1;
            const uint32_t got = __ballot_sync(0xffffffffu, index >= 0), bar = bars + 8 * (kCmRawFull + buf);
            if (lane < kUnits) sts_u32(smem0 + S::kIndex + ((i & 15) * kUnits + lane) * 4, static_cast<uint32_t>(index));
            __syncwarp();
            if (lane == 0) {
                sts_u32(smem0 + S::kMisc + buf * 4, got);
                if (got) mbar_arrive_expect_tx(bar, __popc(got) * kv_unit_bytes(D));
                else mbar_arrive(bar);
            }
            __syncwarp();
            copy_units<D>(c, smem0 + S::kRaw + buf * S::kRawBytes, index, got, lane, bar);
            if (i + 1 < n) at.next(p, c.n_seqs, u0 + i + 1);
        }
        for (int j = max(asked - 4, 0); j < asked; ++j) mbar_wait_bounded(bars + 8 * (kCmRawFull + (j & 3)), (j >> 2) & 1);
    }
    tm_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        tm_after_sync();
        tm_dealloc(tm, kTmCols);
    }
}

constexpr int kTmWarps = 8;

__global__ void __launch_bounds__(32 * kTmWarps) kv_tile_mass_kernel(const KvAttendArgs a, const float* sums, const long long lines) {
    extern __shared__ char dyn[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_rt = a.n_rt;
    const KvView& c = a.c;
    pdl_launch_dependents();
    pdl_wait();
    const Plan p = make_plan<32 * kTmWarps>(c, a.jobs, gridDim.x * kTmWarps, dyn, nullptr);
    const long long w = static_cast<long long>(blockIdx.x) * kTmWarps + warp, u0 = p.runs.start(w);
    const int n = static_cast<int>(p.runs.start(w + 1) - u0);
    if (n == 0) return;
    StepAt at = step_at(p, c.n_seqs, u0);
    constexpr int B = 4;  // steps at once: their pages, then their sums
    for (int i0 = 0; i0 < n; i0 += B) {
        long long line[B];
        float was[B], add[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int slot = at.step * kStep + lane, page = i0 + i < n && slot < at.len ? kv_page(c, at.b, slot) : -1;
            line[i] = page >= 0 ? static_cast<long long>(kv_line(c, page, at.job) + slot % c.page_size) : -1;
            if (++at.step == steps_of(at.len) && i0 + i + 1 < n) at = step_at(p, c.n_seqs, u0 + i0 + i + 1);
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            was[i] = line[i] >= 0 ? ld_l2(c.mass + line[i]) : 0.f;
            add[i] = 0.f;
        }
#pragma unroll 2
        for (int rt = 0; rt < n_rt; ++rt)
#pragma unroll
            for (int i = 0; i < B; ++i) add[i] += line[i] >= 0 ? ld_l2(sums + rt * lines + line[i]) : 0.f;
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (line[i] >= 0) c.mass[line[i]] = was[i] + add[i];
    }
}

int chunk_ctas(const DeviceInfo& di) { return di.sm_count < kChunkCtas ? di.sm_count : kChunkCtas; }

template <int D>
dq_status_t chunk(KvAttendArgs& a, cudaStream_t stream) {
    DeviceInfo di;
    dq_status_t st = device_info(&di);
    if (st != DQ_OK) return st;
    const int ctas = chunk_ctas(di), smem = plan_bytes(a.c.n_seqs) + 1024 + CkSmem<D>::kTotal;
    if ((st = allow_smem(kv_chunk_kernel<D>, smem)) != DQ_OK) return st;
    if ((st = launch_pdl(kv_chunk_kernel<D>, dim3(ctas), kCkThreads, smem, stream, 1, a)) != DQ_OK) return st;
    const long long items = static_cast<long long>(a.c.n_seqs) * a.tokens * a.c.heads * a.group;
    return launch_pdl(kv_chunk_combine_kernel<D>, dim3(static_cast<unsigned>((items + kCcWarps - 1) / kCcWarps)), 32 * kCcWarps, 0,
                      stream, 1, a, ctas);
}

template <int D>
dq_status_t chunk_mass(KvAttendArgs& a, float* sums, cudaStream_t stream) {
    DeviceInfo di;
    dq_status_t st = device_info(&di);
    if (st != DQ_OK) return st;
    const int ctas = chunk_ctas(di), plan = plan_bytes(a.c.n_seqs), smem = plan + 1024 + CmSmem<D>::kTotal;
    const long long lines = static_cast<long long>(a.c.n_pages) * a.c.heads * a.c.page_size;
    if ((st = allow_smem(kv_chunk_mass_kernel<D>, smem)) != DQ_OK) return st;
    const int tiles = a.n_rt;
    if (tiles > 1 && sums) {
        if ((st = launch_pdl(kv_chunk_mass_kernel<D>, dim3(ctas), kCkThreads, smem, stream, 1, a, sums, lines, 0)) != DQ_OK) return st;
        a.jobs = Div(a.c.heads);
        return launch_pdl(kv_tile_mass_kernel, dim3(di.sm_count * 4), 32 * kTmWarps, plan, stream, 1, a, sums, lines);
    }
    a.n_rt = Div(1);
    a.jobs = Div(a.c.heads);
    for (int rt = 0; rt < tiles && st == DQ_OK; ++rt)
        st = launch_pdl(kv_chunk_mass_kernel<D>, dim3(ctas), kCkThreads, smem, stream, 1, a, sums, lines, rt);
    return st;
}

// The jobs of tiles of 128 rows.
void tile_jobs(KvAttendArgs& a) {
    a.n_rt = Div((a.tokens * a.group + kTile - 1) / kTile);
    a.jobs = Div(a.c.heads * a.n_rt);
}

}  // namespace

size_t kv_chunk_part_rows() { return static_cast<size_t>(kChunkCtas) * 2 * kTile; }

dq_status_t launch_kv_chunk(KvAttendArgs a, int head_dim, cudaStream_t stream) {
    tile_jobs(a);
    return head_dim == 128 ? chunk<128>(a, stream) : chunk<64>(a, stream);
}

dq_status_t launch_kv_chunk_mass(KvAttendArgs a, int head_dim, float* sums, cudaStream_t stream) {
    tile_jobs(a);
    return head_dim == 128 ? chunk_mass<128>(a, sums, stream) : chunk_mass<64>(a, sums, stream);
}

dq_status_t read_kv_chunk_error(uint32_t* word, bool clear) {
    unsigned int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_kv_chunk_error, sizeof(v));
    if (e == cudaSuccess && clear && v) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_kv_chunk_error, &zero, sizeof(zero));
    }
    if (e != cudaSuccess) { set_cuda_error(e); return DQ_ERR_CUDA; }
    *word = v;
    return DQ_OK;
}

}  // namespace dq
