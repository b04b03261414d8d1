// dq_kv.cuh -- layout of the paged 4-bit KV cache, shared by the append / evict
// kernels (dq_kv.cu) and the attention kernels (dq_kv_attend.cu).
//
// One unit holds 16 consecutive slots of one KV head, head_dim D = 64 or 128:
//   K       16 rows of D/2 bytes, each a packed row of the framework's INT4
//           format (column 2j in the low nibble of byte j)
//   V       8 slot pairs x D/4 column quads x (even slot, odd slot) x 2 bytes: a
//           32-bit word holds four columns of two neighbouring slots, so that
//           one lop3 gives the f16 pair (slot 2i, slot 2i + 1) of a column --
//           the pair an MMA operand of the P V product needs
//   params  16 x (K scale, K zero, V scale, V zero), FP16
// 16 D + 128 bytes, a multiple of 128, so a unit is one bulk copy.
#pragma once

#include "dq_common.cuh"
#include "dq_internal.h"

namespace dq {

constexpr int kKvTokens = 16;       // slots of one unit
constexpr uint32_t kKvErrPage = 1u; // a page index outside the pool
constexpr uint32_t kKvErrLen = 2u;  // a length or count outside the sequence's pages
constexpr uint32_t kKvErrWait = 4u; // a bounded wait for the kernel's own copies gave up

__host__ __device__ constexpr int kv_unit_bytes(int d) { return kKvTokens * d + kKvTokens * 8; }
__host__ __device__ constexpr int kv_v_offset(int d) { return kKvTokens * d / 2; }
__host__ __device__ constexpr int kv_param_offset(int d) { return kKvTokens * d; }

// Division of 0 <= n < 2^31 by a launch constant: n / d = (umulhi(n, mul) + n) >> shift with
// mul = floor(2^32 (2^shift - d) / d) + 1 and shift = ceil(log2 d).  A handful of cycles where the division by a
// variable is dozens of dependent instructions, in code that a single warp waits for.
struct Div {
    int d = 1;
    uint32_t mul = 1, shift = 0;
    Div() = default;
    explicit Div(int v) : d(v) {
        while ((1u << shift) < static_cast<uint32_t>(v)) ++shift;
        mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - static_cast<uint64_t>(v))) / static_cast<uint64_t>(v) + 1);
    }
    __host__ __device__ operator int() const { return d; }
};
__device__ __forceinline__ int operator/(int n, const Div& d) {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), d.mul) + static_cast<uint32_t>(n)) >> d.shift);
}
__device__ __forceinline__ int operator%(int n, const Div& d) { return n - (n / d) * d.d; }

// dq_kv_cache_t as the kernels take it (validated).
struct KvView {
    uint8_t* units;
    float* mass;
    int32_t* pos;
    int32_t* lengths;
    int32_t* evicted;
    const int32_t* table;
    uint32_t* arrivals;
    int n_seqs, n_pages, max_pages, heads;
    Div page_size;
};

inline KvView kv_view(const dq_kv_cache_t& c) {
    return KvView{c.units, c.mass, c.pos, c.lengths, c.evicted, c.page_table, c.arrivals,
                  c.n_seqs, c.n_pages, c.max_pages, c.kv_heads, Div(c.page_size)};
}

// Loads from L2 of what earlier kernels or other CTAs wrote.  They keep the order of the source: those that are to be
// in flight at once stand together there, before the first use of any.
__device__ __forceinline__ int ld_l2(const int* p) { return __ldcg(p); }
__device__ __forceinline__ uint32_t ld_l2(const uint32_t* p) { return __ldcg(p); }
__device__ __forceinline__ float ld_l2(const float* p) { return __ldcg(p); }
__device__ __forceinline__ uint4 ld_l2_v4(const void* p) { return __ldcg(static_cast<const uint4*>(p)); }

// The page of a slot, or -1 where the table has none inside the pool.
__device__ __forceinline__ int kv_page(const KvView& c, int b, int slot) {
    const int p = ld_l2(c.table + static_cast<size_t>(b) * c.max_pages + slot / c.page_size);
    return (p >= 0 && p < c.n_pages) ? p : -1;
}

// Index of (page, head, offset 0) in mass / pos, and of its first unit.
__device__ __forceinline__ size_t kv_line(const KvView& c, int page, int h) {
    return (static_cast<size_t>(page) * c.heads + h) * c.page_size;
}

template <int D>
__device__ __forceinline__ uint8_t* kv_unit(const KvView& c, int page, int h, int off) {
    return c.units + (kv_line(c, page, h) + off) / kKvTokens * kv_unit_bytes(D);
}

// Tokens of sequence b, kept inside its pages.
__device__ __forceinline__ int kv_length(const KvView& c, int b, bool* bad) {
    const int n = ld_l2(c.lengths + b), cap = c.max_pages * c.page_size;
    if (n < 0 || n > cap) *bad = true;
    return n < 0 ? 0 : (n > cap ? cap : n);
}

// A launch as a programmatic dependent of the preceding work on the stream, in clusters of cluster x 1 CTAs.
template <class K, class... A>
inline dq_status_t launch_pdl(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, int cluster, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { set_cuda_error(e); return DQ_ERR_CUDA; }
    return DQ_OK;
}

}  // namespace dq
