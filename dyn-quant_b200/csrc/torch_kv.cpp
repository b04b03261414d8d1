// torch_kv.cpp -- the paged 4-bit KV cache in dyn_quant._C: class KVCache, the
// checked handle behind dyn_quant.kv_cache.Int4KVCache, over the C ABI's
// dq_kv_* calls.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <array>
#include <vector>

#include "../../include/dq_abi.h"

namespace {

void check_status(dq_status_t s, const char* what) {
    if (s == DQ_OK) return;
    if (s == DQ_ERR_CUDA)
        TORCH_CHECK(false, what, " failed: ", dq_status_string(s), " (cudaError ", dq_last_cuda_error(), ")");
    TORCH_CHECK(false, what, " failed: ", dq_status_string(s));
}

// The cache's tensors, checked once; each call then checks its own arguments
// only.  Holds references to the tensors whose addresses it keeps.
class KVCache {
public:
    KVCache(const torch::Tensor& units, const torch::Tensor& mass, const torch::Tensor& pos,
            const torch::Tensor& lengths, const torch::Tensor& evicted, const torch::Tensor& page_table,
            const torch::Tensor& arrivals)
        : keep_{units, mass, pos, lengths, evicted, page_table, arrivals} {
        TORCH_CHECK(units.is_cuda() && units.is_contiguous() && units.scalar_type() == at::kByte && units.dim() == 4,
                    "units must be a contiguous CUDA uint8 tensor [n_pages, kv_heads, page_size / 16, unit bytes]");
        const int64_t ub = units.size(3);
        TORCH_CHECK(ub == static_cast<int64_t>(dq_kv_unit_bytes(64)) || ub == static_cast<int64_t>(dq_kv_unit_bytes(128)),
                    "head_dim must be 64 or 128");
        dev_ = units.device();
        const int64_t pages = units.size(0), heads = units.size(1), page = units.size(2) * 16;
        auto check = [&](const torch::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape) {
            TORCH_CHECK(t.device() == dev_, name, " must be on the same device as units");
            TORCH_CHECK(t.is_contiguous() && t.scalar_type() == type && t.sizes() == shape, name,
                        " must be a contiguous ", type, " tensor of shape ", shape);
        };
        check(mass, "mass", at::kFloat, {pages, heads, page});
        check(pos, "pos", at::kInt, {pages, heads, page});
        TORCH_CHECK(lengths.dim() == 1 && page_table.dim() == 2, "lengths must be 1D and page_table 2D");
        const int64_t seqs = lengths.size(0);
        TORCH_CHECK(seqs <= 1024, "at most 1024 sequences per cache");
        check(lengths, "lengths", at::kInt, {seqs});
        check(evicted, "evicted", at::kInt, {seqs});
        check(arrivals, "arrivals", at::kInt, {seqs * (1 + heads)});
        check(page_table, "page_table", at::kInt, {seqs, page_table.size(1)});
        TORCH_CHECK(pages <= INT32_MAX && heads <= 65535 && page_table.size(1) * page <= (int64_t{1} << 30),
                    "cache too large");
        c_.units = static_cast<uint8_t*>(units.data_ptr());
        c_.mass = mass.data_ptr<float>();
        c_.pos = pos.data_ptr<int32_t>();
        c_.lengths = lengths.data_ptr<int32_t>();
        c_.evicted = evicted.data_ptr<int32_t>();
        c_.page_table = page_table.data_ptr<int32_t>();
        c_.arrivals = reinterpret_cast<uint32_t*>(arrivals.data_ptr<int32_t>());
        c_.n_seqs = static_cast<int32_t>(seqs);
        c_.n_pages = static_cast<int32_t>(pages);
        c_.max_pages = static_cast<int32_t>(page_table.size(1));
        c_.page_size = static_cast<int32_t>(page);
        c_.kv_heads = static_cast<int32_t>(heads);
        c_.head_dim = static_cast<int32_t>((ub - 128) / 16);
    }

    // k, v [n_seqs, T, kv_heads, head_dim] or [n_seqs, kv_heads, head_dim] (T = 1)
    py::object append(const torch::Tensor& k_in, const torch::Tensor& v_in, const c10::optional<torch::Tensor>& counts,
                      const c10::optional<torch::Tensor>& at, bool values) {
        const at::cuda::CUDAGuard guard(dev_);
        const torch::Tensor k = rows(k_in, "k", c_.kv_heads), v = rows(v_in, "v", c_.kv_heads);
        TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
        const int32_t tokens = static_cast<int32_t>(k.size(1));
        const int32_t* cn = per_seq(counts, "counts");
        const int32_t* start = per_seq(at, "at");
        torch::Tensor kv, vv;
        if (values) {
            kv = torch::empty(k.sizes(), k.options());
            vv = torch::empty(k.sizes(), k.options());
        }
        int64_t ks[3], vs[3];
        strides(k, ks);
        strides(v, vs);
        check_status(dq_kv_append(&c_, h16(k), ks, h16(v), vs, tokens, cn, start, values ? h16(kv) : nullptr,
                                  values ? h16(vv) : nullptr, stream()),
                     "kv append");
        if (!values) return py::none();
        return py::make_tuple(kv.view(k_in.sizes()), vv.view(k_in.sizes()));
    }

    // q [n_seqs, T, q_heads, head_dim] or [n_seqs, q_heads, head_dim] -> out of q's shape (and lse)
    py::object attend(const torch::Tensor& q_in, double scale, const c10::optional<torch::Tensor>& counts,
                      bool accumulate, const c10::optional<torch::Tensor>& out_in, bool return_lse) {
        const at::cuda::CUDAGuard guard(dev_);
        const torch::Tensor q = rows(q_in, "q", 0);
        dq_kv_attend_t r{};
        r.tokens = static_cast<int32_t>(q.size(1));
        r.q_heads = static_cast<int32_t>(q.size(2));
        TORCH_CHECK(r.q_heads > 0 && r.q_heads % c_.kv_heads == 0, "q heads must be a multiple of the cache's ",
                    c_.kv_heads, " KV heads, got ", r.q_heads);
        r.counts = per_seq(counts, "counts");
        torch::Tensor out;
        if (out_in.has_value() && out_in->defined()) {
            TORCH_CHECK(out_in->device() == dev_ && out_in->scalar_type() == at::kHalf && out_in->sizes() == q_in.sizes(),
                        "out must be a float16 tensor of q's shape on the cache's device");
            out = out_in->dim() == 3 ? out_in->unsqueeze(1) : *out_in;
            TORCH_CHECK(direct(out), "out needs head_dim contiguous, strides multiples of 8 and a 16-byte aligned start");
            TORCH_CHECK(apart(out), "out must not overlap itself");
            TORCH_CHECK(!meet(out, q), "out must not lie among q's rows: rows are read after others are written");
        } else {
            out = torch::empty({q.size(0), q.size(1), q.size(2), q.size(3)}, q.options());
        }
        torch::Tensor lse;
        if (return_lse) lse = torch::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
        r.q = h16(q);
        r.out = h16(out);
        strides(q, r.q_stride);
        strides(out, r.out_stride);
        r.lse = return_lse ? lse.data_ptr<float>() : nullptr;
        r.scale = static_cast<float>(scale);
        r.accumulate = accumulate ? 1 : 0;
        const size_t need = dq_kv_attend_workspace_bytes(&c_, r.tokens, r.q_heads, r.accumulate);
        auto ws = scratch(need);
        check_status(dq_kv_attend(&c_, &r, ws.data_ptr(), need, stream()), "kv attend");
        if (!(out_in.has_value() && out_in->defined())) out = out.view(q_in.sizes());
        else out = *out_in;
        if (!return_lse) return py::cast(out);
        return py::make_tuple(out, q_in.dim() == 3 ? lse.squeeze(1) : lse);
    }

    void evict(int64_t keep, int64_t recent, int64_t sink) {
        TORCH_CHECK(keep >= 1 && keep <= INT32_MAX && recent >= 0 && sink >= 0 && recent <= keep && sink <= keep - recent,
                    "evict needs keep >= 1 and recent + sink <= keep, got keep=", keep, " recent=", recent, " sink=", sink);
        const at::cuda::CUDAGuard guard(dev_);
        const size_t need = dq_kv_evict_workspace_bytes(&c_, static_cast<int32_t>(keep));
        auto ws = scratch(need);
        check_status(dq_kv_evict(&c_, static_cast<int32_t>(keep), static_cast<int32_t>(recent), static_cast<int32_t>(sink),
                                 ws.data_ptr(), need, stream()),
                     "kv evict");
    }

private:
    static uint16_t* h16(const torch::Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }
    void* stream() const { return at::cuda::getCurrentCUDAStream(dev_.index()).stream(); }
    torch::Tensor scratch(size_t bytes) const {
        return torch::empty({static_cast<int64_t>(bytes)}, torch::TensorOptions().dtype(torch::kUInt8).device(dev_));
    }
    static void strides(const torch::Tensor& t, int64_t s[3]) {
        // the stride of a dimension of one is never used
        for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    }
    // Whether the kernels can read or write it in place.
    static bool direct(const torch::Tensor& t) {
        if (t.stride(3) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u)) return false;
        for (int i = 0; i < 3; ++i)
            if (t.size(i) > 1 && t.stride(i) % 8 != 0) return false;
        return true;
    }
    // No two rows of it share memory.
    static bool apart(const torch::Tensor& t) {
        std::array<int, 3> d{0, 1, 2};
        std::sort(d.begin(), d.end(), [&](int a, int b) { return t.stride(a) < t.stride(b); });
        int64_t extent = t.size(3);
        for (int i : d) {
            if (t.size(i) <= 1) continue;
            if (t.stride(i) < extent) return false;
            extent = (t.size(i) - 1) * t.stride(i) + extent;
        }
        return true;
    }
    // Whether the memory between two tensors' first and last values overlaps.
    static bool meet(const torch::Tensor& a, const torch::Tensor& b) {
        if (a.numel() == 0 || b.numel() == 0) return false;
        auto end = [](const torch::Tensor& t) {
            int64_t last = 0;
            for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
            return h16(t) + last + 1;
        };
        return h16(a) < end(b) && h16(b) < end(a);
    }
    // [n_seqs, T, heads, head_dim] float16, readable in place (heads 0: any number)
    torch::Tensor rows(const torch::Tensor& t_in, const char* name, int64_t heads) const {
        TORCH_CHECK(t_in.is_cuda() && t_in.device() == dev_, name, " must be on the cache's device ", dev_);
        TORCH_CHECK(t_in.is_floating_point(), name, " must be a floating-point tensor");
        TORCH_CHECK(t_in.dim() == 3 || t_in.dim() == 4, name, " must be [n_seqs, T, heads, head_dim] or [n_seqs, heads, head_dim]");
        torch::Tensor t = t_in.dim() == 3 ? t_in.unsqueeze(1) : t_in;
        TORCH_CHECK(t.size(0) == c_.n_seqs && t.size(3) == c_.head_dim && (heads == 0 || t.size(2) == heads), name,
                    " does not fit the cache: n_seqs=", c_.n_seqs, " head_dim=", c_.head_dim, " kv_heads=", c_.kv_heads,
                    ", got ", t_in.sizes());
        TORCH_CHECK(t.size(1) <= INT32_MAX && t.size(2) <= INT32_MAX && t.size(1) * t.size(2) <= (int64_t{1} << 26), name,
                    " has too many rows");
        if (t.scalar_type() != at::kHalf) t = t.to(at::kHalf);
        if (t.numel() && !direct(t)) t = t.contiguous();
        if (t.numel() && !direct(t)) t = t.clone();  // a contiguous view that starts off a 16-byte boundary
        return t;
    }
    const int32_t* per_seq(const c10::optional<torch::Tensor>& t, const char* name) const {
        if (!t.has_value() || !t->defined()) return nullptr;
        TORCH_CHECK(t->device() == dev_ && t->scalar_type() == at::kInt && t->is_contiguous() && t->dim() == 1 &&
                        t->size(0) == c_.n_seqs,
                    name, " must be a contiguous int32 tensor [n_seqs] on the cache's device");
        return t->data_ptr<int32_t>();
    }

    std::vector<torch::Tensor> keep_;
    dq_kv_cache_t c_{};
    torch::Device dev_{torch::kCPU};
};

}  // namespace

void bind_kv(py::module_& m) {
    py::class_<KVCache>(m, "KVCache")
        .def(py::init<const torch::Tensor&, const torch::Tensor&, const torch::Tensor&, const torch::Tensor&,
                      const torch::Tensor&, const torch::Tensor&, const torch::Tensor&>(),
             py::arg("units"), py::arg("mass"), py::arg("pos"), py::arg("lengths"), py::arg("evicted"),
             py::arg("page_table"), py::arg("arrivals"))
        .def("append", &KVCache::append, py::arg("k"), py::arg("v"), py::arg("counts"), py::arg("at"), py::arg("values"))
        .def("attend", &KVCache::attend, py::arg("q"), py::arg("scale"), py::arg("counts"), py::arg("accumulate"),
             py::arg("out"), py::arg("return_lse"))
        .def("evict", &KVCache::evict, py::arg("keep"), py::arg("recent"), py::arg("sink"));
}
