// dq_kv_plan.cuh -- what the attention kernels over the 4-bit KV cache share:
// their arguments, the split of the work into equal runs (on the device, from
// the lengths), the exchange of partial results, and small arithmetic.
#pragma once

#include <cfloat>

#include "dq_kv.cuh"

namespace dq {

struct KvAttendArgs {
    KvView c;
    const uint16_t* q;
    uint16_t* out;
    long long qs[3], os[3];  // strides in values: sequence, token, head
    float* lse;              // [n_seqs][tokens][q_heads] natural log, or null
    float* lse2;             // workspace: the same in log2 (mass pass), or null
    float* scores;           // workspace: [units of the pool][16][pitch] scores in log2 for the mass pass, or null
    int pitch;               // rows of a KV head, rounded up to 1, 2, 4 or 8
    const int32_t* counts;
    float* part;             // [CTAs][2][rows][D]
    float* part_ml;          // [CTAs][2][rows][2]
    float* first;            // [warps][rows][D + 2] pieces of jobs that end inside a run
    int* pre;                // [n_seqs + 1] the plan's prefix sums, for the combining kernel
    uint32_t* done;          // [n_seqs][heads] CTAs of a cut job that have arrived (one row tile)
    int tokens;              // query tokens
    Div group, n_rt, jobs;   // query heads per KV head, row tiles, jobs of a sequence
    float scale2;            // scale * log2(e), times 2^14 where the codes are c 2^-14
    int depth;               // ring slots per warp
    int first_off, places;   // shared memory for some of those pieces: its offset, how many
};

// Attention of many query rows per KV head (dq_kv_chunk.cu): workspace rows, and the launch (a's lse2 filled in too).
constexpr int kChunkRows = 128;  // query rows of a tile
size_t kv_chunk_part_rows();     // rows of part / part_ml
dq_status_t launch_kv_chunk(KvAttendArgs a, int head_dim, cudaStream_t stream);
// The mass pass for any number of rows, from lse2.  sums: [row tiles][n_pages][kv_heads][page_size], or null.
dq_status_t launch_kv_chunk_mass(KvAttendArgs a, int head_dim, float* sums, cudaStream_t stream);

namespace {

constexpr float kNone = -FLT_MAX;     // running maximum of a row that has seen no key
constexpr float kLazy = 8.0f;         // a score passes the running maximum by this much (log2) before it moves
constexpr int kStep = 2 * kKvTokens;  // slots of one step of a run

// The list of steps: a job is steps_of(len[b]) steps of one (sequence, KV head,
// row tile), a sequence has `jobs` of them one after another, pre[b] counts the
// steps of one job of every sequence before b.  Warp w takes base steps, one
// more if w < rem.  Short lists are cut into runs of up to 4 steps rather than
// one: a job then needs fewer warps, and its pieces meet in one CTA.
// a / b for 0 <= a, 0 < b, with the short division where it does.
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return ((a | b) >> 31) == 0 ? static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
__device__ __forceinline__ int quotient(long long a, const Div& b) {
    return (a >> 31) == 0 ? static_cast<int>(a) / b : static_cast<int>(a / b.d);
}

struct Runs {
    long long base, total;
    int rem;

    __device__ __forceinline__ Runs() {}
    __device__ __forceinline__ Runs(int job_steps, int n_seqs, int jobs, int warps) {
        total = static_cast<long long>(job_steps) * jobs;
        const int least = min(4, (job_steps + n_seqs - 1) / n_seqs);
        if (total < static_cast<long long>(warps) * least) warps = max(1, static_cast<int>(total) / max(least, 1));
        base = quotient(total, warps);
        rem = static_cast<int>(total - base * warps);
    }
    __device__ __forceinline__ long long start(long long w) const {
        return min(w * base + (w < rem ? w : rem), total);
    }
    // the warp whose run has step u
    __device__ __forceinline__ long long warp_of(long long u) const {
        const long long cut = rem * (base + 1);
        return u < cut ? quotient(u, base + 1) : rem + quotient(u - cut, base);
    }
};

struct Plan {
    const int* pre;
    const int* len;
    Div jobs;
    Runs runs;
};

template <int S = kStep>
__host__ __device__ inline int steps_of(int len) {
    return (len + S - 1) / S;
}

// Bytes of the plan in shared memory.
__host__ __device__ inline int plan_bytes(int n_seqs) { return ((2 * n_seqs + 1) * 4 + 127) / 128 * 128; }

// Built by every CTA from the lengths (a few KB from L2); all threads call it.
template <int NT, int S = kStep>
__device__ Plan make_plan(const KvView& c, const Div& jobs, int warps, char* smem, unsigned int* err) {
    int* pre = reinterpret_cast<int*>(smem);
    int* lens = pre + c.n_seqs + 1;
    __shared__ int wtot[NT / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int run = 0;
    for (int b0 = 0; b0 < c.n_seqs; b0 += NT) {
        const int b = b0 + tid;
        int v = 0;
        if (b < c.n_seqs) {
            bool bad = false;
            const int n = kv_length(c, b, &bad);
            if (bad && err) atomicOr(err, kKvErrLen);
            lens[b] = n;
            v = steps_of<S>(n);
        }
        int inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        if (lane == 31) wtot[warp] = inc;
        __syncthreads();
        int before = run;
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
    p.jobs = jobs;
    p.runs = Runs(run, c.n_seqs, jobs, warps);
    return p;
}

// Where a step lies: sequence, its length, job and step of the job.
struct StepAt {
    int b, len, job, step;
};

__device__ __forceinline__ StepAt step_at(const Plan& p, int n_seqs, long long u) {
    const int v = quotient(u, p.jobs);  // pre[b] <= v < pre[b + 1]: the last b with pre[b] <= v
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.pre[mid] <= v) lo = mid;
        else hi = mid;
    }
    const int st = p.pre[lo + 1] - p.pre[lo];
    const long long r = u - static_cast<long long>(p.pre[lo]) * p.jobs;
    StepAt a;
    a.b = lo;
    a.len = p.len[lo];
    a.job = static_cast<int>(quotient(r, static_cast<long long>(st)));
    a.step = static_cast<int>(r - static_cast<long long>(a.job) * st);
    return a;
}

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Two FP32 operations in one instruction, on the pair of a lane's rows 2t, 2t + 1.
struct f2 {
    unsigned long long v;
    __device__ __forceinline__ f2() {}
    __device__ __forceinline__ f2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
    __device__ __forceinline__ explicit f2(float x) : f2(x, x) {}
    __device__ __forceinline__ float x() const {
        return __uint_as_float(static_cast<uint32_t>(v));
    }
    __device__ __forceinline__ float y() const {
        return __uint_as_float(static_cast<uint32_t>(v >> 32));
    }
};
__device__ __forceinline__ f2 operator+(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f2 operator*(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

__device__ __forceinline__ uint32_t pack_f32(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 1 / sum of a row's weights; 0 where it has seen no key, not a number where the sum is not.
__device__ __forceinline__ float row_norm(float sum) {
    return sum > 0.f ? __fdividef(1.f, sum) : (sum == 0.f ? 0.f : sum);  // sum <= 2^38: weights of 2^8, 2^30 slots
}

// lse of a row, in log2 and natural.
__device__ __forceinline__ void store_lse(const KvAttendArgs& a, int b, int tok, int head, float m, float sum) {
    const size_t i = (static_cast<size_t>(b) * a.tokens + tok) * (a.c.heads * a.group) + head;
    const float l2 = sum == 0.f ? -INFINITY : m + __log2f(sum);  // absolute error 2^-21
    if (a.lse) a.lse[i] = l2 * 0.693147180559945309f;
    if (a.lse2) a.lse2[i] = l2;
}

// Columns col .. col + N - 1 of row r of KV head h, normalised; the thread with column 0 stores the row's lse.
template <int N>
__device__ __forceinline__ void store_row(const KvAttendArgs& a, int b, int h, int r, int col, const float (&v)[N], float m,
                                          float sum) {
    const int tok = r / a.group, head = h * a.group + r - tok * a.group;
    const float f = row_norm(sum);
    uint16_t* dst = a.out + b * a.os[0] + tok * a.os[1] + head * a.os[2] + col;
#pragma unroll
    for (int i = 0; i < N; i += 8)
        *reinterpret_cast<uint4*>(dst + i) =
            make_uint4(pack_f32(v[i] * f, v[i + 1] * f), pack_f32(v[i + 2] * f, v[i + 3] * f),
                       pack_f32(v[i + 4] * f, v[i + 5] * f), pack_f32(v[i + 6] * f, v[i + 7] * f));
    if (col == 0) store_lse(a, b, tok, head, m, sum);
}

// The CTAs that share a job (c0 .. c0 + n - 1) and the workspace slot of the first; every later CTA begins
// inside the job, which is its slot 0.
struct Share {
    long long c0;
    int n, slot0;
};

template <int W>
__device__ __forceinline__ Share share_of(const int* pre, int n_seqs, const Div& jobs, const Runs& runs, int b, int job) {
    Share s{0, 0, 0};
    const int p0 = pre[b], ul = pre[b + 1] - p0;
    if (ul == 0) return s;
    const long long u0 = static_cast<long long>(p0) * jobs + static_cast<long long>(ul) * job;
    s.c0 = runs.warp_of(u0) / W;
    s.n = static_cast<int>(runs.warp_of(u0 + ul - 1) / W - s.c0) + 1;
    const long long start = runs.start(s.c0 * W);
    if (s.n > 1 && u0 > start) {
        // the job at the CTA's start has slot 0 if the border cuts it
        const int v = quotient(start, jobs);
        int lo = 0, hi = b + 1;  // pre[lo] <= v < pre[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= v) lo = mid;
            else hi = mid;
        }
        const long long in = start - static_cast<long long>(pre[lo]) * jobs, st = pre[lo + 1] - pre[lo];
        s.slot0 = in != quotient(in, st) * st ? 1 : 0;
    }
    return s;
}

// One warp joins row r's partial sums: maxima and sums a lane each, then the outputs N partials at a time (eight where
// a job is cut between many warps; four leave room for all of dq_kv_chunk.cu's rows at once: 9 us for 10).
template <int D, int NT, int N = 8>
__device__ __forceinline__ void join_row(const KvAttendArgs& a, const Share& s, int b, int h, int rt, int r) {
    constexpr int R = 8 * NT, V = D / 32;  // V columns of a lane, side by side; N partials at a time
    const int lane = threadIdx.x & 31, rl = r - rt * R, first = s.slot0 * R;  // only the first CTA's may be its slot 1
    const size_t row0 = static_cast<size_t>(s.c0) * 2 * R + rl;
    const float2* ml0 = reinterpret_cast<const float2*>(a.part_ml) + row0;
    const float* o0 = a.part + row0 * D + V * lane;
    auto ml_at = [&](int i) { return i < s.n ? __ldcg(ml0 + (i == 0 ? first : i * 2 * R)) : make_float2(kNone, 0.f); };
    float x[N][V];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float* src = o0 + static_cast<size_t>(i0) * 2 * R * D + j * 2 * R * D + (i0 + j == 0 ? first * D : 0);
            const bool on = i0 + j < s.n;
            if constexpr (V == 4) {
                const float4 y = on ? __ldcg(reinterpret_cast<const float4*>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[j][0] = y.x; x[j][1] = y.y; x[j][2] = y.z; x[j][3] = y.w;
            } else {
                const float2 y = on ? __ldcg(reinterpret_cast<const float2*>(src)) : make_float2(0.f, 0.f);
                x[j][0] = y.x; x[j][1] = y.y;
            }
        }
    };
    float2 ml = ml_at(lane);
    fetch(0);
    float m = ml.x, sum = 0.f, v[V];
    for (int i = lane + 32; i < s.n; i += 32) m = fmaxf(m, ml_at(i).x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
#pragma unroll 1
    for (int i0 = 0; i0 < s.n; i0 += N) {
        if (i0 > 0 && i0 % 32 == 0) ml = ml_at(i0 + lane);
        const float f = ml.x > kNone ? ex2(ml.x - m) : (ml.x == kNone ? 0.f : ml.x);
        if (i0 % 32 == 0) sum += ml.y * f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float fj = __shfl_sync(0xffffffffu, f, i0 % 32 + j);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = fmaf(x[j][k], fj, v[k]);
        }
        if (i0 + N < s.n) fetch(i0 + N);
    }
    sum = warp_sum(sum);
    const int tok = r / a.group, head = h * a.group + r - tok * a.group;
    const float f = row_norm(sum);
    uint16_t* dst = a.out + b * a.os[0] + tok * a.os[1] + head * a.os[2] + V * lane;
#pragma unroll
    for (int k = 0; k < V; k += 2) *reinterpret_cast<uint32_t*>(dst + k) = pack_f32(v[k] * f, v[k + 1] * f);
    if (lane == 0) store_lse(a, b, tok, head, m, sum);
}

template <class K>
dq_status_t allow_smem(K kernel, int smem) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { set_cuda_error(e); return DQ_ERR_CUDA; }
    return DQ_OK;
}

}  // namespace

}  // namespace dq
