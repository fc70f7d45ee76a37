// Python binding of the operator API's success path on torch tensors (the
// role of the reference's pybind `forward` / `forward_into`,
// kernels/int4gemv/bindings.cpp:145-176 and kernels/qgemv/bindings.cpp:66-115).
//
// It makes the checks of the Python wrapper's success predicate
// (ext.py `_fast_ok`) on the tensors' metadata in C++, then calls the C ABI
// (cl_int4gemv_ex / cl_qgemv_ex) on the current stream of the tensors'
// device.  When a check fails, or the C ABI reports an error, it returns a
// nonzero code without raising, and the Python wrapper runs its ordered
// checks, which raise the reference's messages.  No computation happens here.
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <array>
#include <cmath>

#include "../../include/cudalab_gemv.h"

namespace {

constexpr int kNotFast = -1000;  // a check of the success predicate failed
constexpr int kInt4 = 0, kInt8 = 1;

bool on(const at::Tensor& t, c10::DeviceIndex d) { return t.is_cuda() && t.get_device() == d; }

// W / scale / x of one GEMV: the success predicate of the Python wrapper
// (INT4: W uint8 [N, K/2] with K % 128 == 0, scale fp16 [N, K/128]; INT8: W
// int8 [N, K], scale fp32 [N]; x fp16 [K]; all contiguous, on W's device).
bool inputs_ok(int kind, const at::Tensor& W, const at::Tensor& s, const at::Tensor& x,
               int64_t& N, int64_t& K) {
    if (!W.is_cuda() || W.dim() != 2 || !W.is_contiguous()) return false;
    N = W.size(0);
    const int64_t cols = W.size(1);
    if (N <= 0 || cols <= 0) return false;
    const c10::DeviceIndex d = W.get_device();
    if (kind == kInt4) {
        if (W.scalar_type() != at::kByte || cols % 64 != 0) return false;
        K = 2 * cols;
        if (s.scalar_type() != at::kHalf || s.dim() != 2 || s.size(0) != N || s.size(1) != cols / 64)
            return false;
    } else {
        if (W.scalar_type() != at::kChar) return false;
        K = cols;
        if (s.scalar_type() != at::kFloat || s.dim() != 1 || s.size(0) != N) return false;
    }
    return s.is_contiguous() && on(s, d) && x.scalar_type() == at::kHalf && x.dim() == 1 &&
           x.size(0) == K && x.is_contiguous() && on(x, d);
}

int launch(int kind, const std::string& variant, const at::Tensor& W, const at::Tensor& s,
           const at::Tensor& x, const at::Tensor& out, int64_t N, int64_t K, uint32_t flags) {
    const c10::DeviceIndex d = W.get_device();
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != d) guard.set_index(d);
    void* st = c10::cuda::getCurrentCUDAStream(d).stream();
    if (kind == kInt4)
        return cl_int4gemv_ex(variant.c_str(), static_cast<const uint8_t*>(W.data_ptr()),
                              s.data_ptr(), x.data_ptr(), out.data_ptr(), N, K, st, flags);
    return cl_qgemv_ex(variant.c_str(), static_cast<const int8_t*>(W.data_ptr()),
                       static_cast<const float*>(s.data_ptr()), x.data_ptr(), out.data_ptr(), N, K,
                       st, flags);
}

// 0 on success; kNotFast or the C ABI's status otherwise (nothing raised).
int forward_into(int kind, const std::string& variant, const at::Tensor& W, const at::Tensor& s,
                 const at::Tensor& x, const at::Tensor& out, int64_t flags) {
    int64_t N = 0, K = 0;
    if (!inputs_ok(kind, W, s, x, N, K)) return kNotFast;
    if (out.scalar_type() != at::kHalf || out.dim() != 1 || out.size(0) != N ||
        !out.is_contiguous() || !on(out, W.get_device()))
        return kNotFast;
    return launch(kind, variant, W, s, x, out, N, K, static_cast<uint32_t>(flags));
}

// The output tensor on success; None otherwise (nothing raised).
c10::optional<at::Tensor> forward(int kind, const std::string& variant, const at::Tensor& W,
                                  const at::Tensor& s, const at::Tensor& x, int64_t flags) {
    int64_t N = 0, K = 0;
    if (!inputs_ok(kind, W, s, x, N, K)) return c10::nullopt;
    at::Tensor out = at::empty({N}, x.options());
    if (launch(kind, variant, W, s, x, out, N, K, static_cast<uint32_t>(flags)) != CL_OK)
        return c10::nullopt;
    return out;
}

// ---- the decode step's attention operators (attention_ext.py): the same
// pattern, the checks of its `_validate` methods as one predicate ----

int type16(const at::Tensor& t) {
    return t.scalar_type() == at::kHalf ? CL_DTYPE_F16
           : t.scalar_type() == at::kBFloat16 ? CL_DTYPE_BF16 : -1;
}

// 16-bit rows [.., dim] with a contiguous last dimension on device d.
bool rows_ok(const at::Tensor& t, int dims, c10::DeviceIndex d) {
    return t.dim() == dims && type16(t) >= 0 && on(t, d) && t.stride(dims - 1) == 1;
}

bool plain_ok(const at::Tensor& t, int dims, at::ScalarType s, c10::DeviceIndex d) {
    return t.dim() == dims && t.scalar_type() == s && t.is_contiguous() && on(t, d);
}

// (bits, page_size) of a cache tensor; false when its form does not fit head_dim.
bool pages_ok(const at::Tensor& p, int64_t head_dim, c10::DeviceIndex d, int32_t* bits,
              int32_t* page_size) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return false;
    if (!plain_ok(p, 4, at::kByte, d) || p.numel() == 0) return false;
    const int64_t bytes = p.size(3);
    if (bytes != 32 * head_dim + 64 && bytes != 16 * head_dim + 64) return false;
    *bits = bytes == 32 * head_dim + 64 ? 8 : 4;
    if (p.size(2) > (1 << 16)) return false;
    *page_size = static_cast<int32_t>(16 * p.size(2));
    return true;
}

void* begin(c10::DeviceIndex d, c10::cuda::OptionalCUDAGuard* guard) {
    if (c10::cuda::current_device() != d) guard->set_index(d);
    return c10::cuda::getCurrentCUDAStream(d).stream();
}

using Pair = std::pair<at::Tensor, at::Tensor>;

// An uninitialised tensor of the caching allocator, without the dispatcher
// (0.3 us less).
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::DeviceIndex d) {
    return at::detail::empty_cuda(sizes, type, c10::Device(c10::DeviceType::CUDA, d), c10::nullopt);
}

int64_t count(at::IntArrayRef sizes) {
    int64_t n = 1;
    for (int64_t s : sizes) n *= s;
    return n;
}

// Two contiguous results of one call in one allocation, which lives as long as
// either (0.7 us less than two allocations, of the 5 us of a small call).  The
// first one's bytes are a multiple of 16, so both are aligned.
Pair empty_two(at::IntArrayRef first, at::ScalarType first_type, at::IntArrayRef second,
               at::ScalarType second_type, c10::DeviceIndex d) {
    const int64_t bytes = count(first) * static_cast<int64_t>(c10::elementSize(first_type));
    const int64_t more = count(second) * static_cast<int64_t>(c10::elementSize(second_type));
    const at::Tensor all = empty({bytes + more}, at::kByte, d);
    auto part = [&](at::IntArrayRef sizes, at::ScalarType type, int64_t at_byte) {
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
            c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
        t.unsafeGetTensorImpl()->set_storage_offset(
            at_byte / static_cast<int64_t>(c10::elementSize(type)));
        return t;
    };
    return Pair(part(first, first_type, 0), part(second, second_type, bytes));
}

c10::optional<Pair> qknorm_rope(const at::Tensor& q, const at::Tensor& k,
                                const c10::optional<at::Tensor>& qw,
                                const c10::optional<at::Tensor>& kw, const at::Tensor& table,
                                const at::Tensor& positions, double eps, bool interleaved) {
    if (!q.is_cuda()) return c10::nullopt;
    const c10::DeviceIndex d = q.get_device();
    if (!rows_ok(q, 3, d) || !rows_ok(k, 3, d) || q.scalar_type() != k.scalar_type() ||
        k.size(0) != q.size(0) || k.size(2) != q.size(2) || q.size(1) <= 0 || k.size(1) <= 0)
        return c10::nullopt;
    const int64_t D = q.size(2);
    if (qw.has_value() != kw.has_value()) return c10::nullopt;
    if (qw && (!plain_ok(*qw, 1, q.scalar_type(), d) || !plain_ok(*kw, 1, q.scalar_type(), d) ||
               qw->size(0) != D || kw->size(0) != D))
        return c10::nullopt;
    const bool wide = positions.scalar_type() == at::kLong;
    if (!plain_ok(table, 2, at::kFloat, d) ||
        !plain_ok(positions, 1, wide ? at::kLong : at::kInt, d) || positions.size(0) != q.size(0))
        return c10::nullopt;
    cl_qknorm_rope_desc desc{};
    desc.tokens = q.size(0);
    desc.table_rows = table.size(0);
    desc.q_token = q.stride(0), desc.q_head = q.stride(1);
    desc.k_token = k.stride(0), desc.k_head = k.stride(1);
    desc.q_out_token = q.size(1) * D, desc.k_out_token = k.size(1) * D;
    desc.q_out_head = desc.k_out_head = D;
    desc.q_heads = static_cast<int32_t>(q.size(1));
    desc.kv_heads = static_cast<int32_t>(k.size(1));
    desc.head_dim = static_cast<int32_t>(D);
    desc.rotary = static_cast<int32_t>(table.size(1));
    desc.interleaved = interleaved;
    desc.positions64 = wide;
    desc.dtype = type16(q);
    desc.eps = static_cast<float>(eps);
    c10::cuda::OptionalCUDAGuard guard;
    void* st = begin(d, &guard);
    Pair out = empty_two(q.sizes(), q.scalar_type(), k.sizes(), k.scalar_type(), d);
    if (cl_qknorm_rope(q.data_ptr(), k.data_ptr(), qw ? qw->data_ptr() : nullptr,
                       kw ? kw->data_ptr() : nullptr, table.data_ptr<float>(),
                       positions.data_ptr(), out.first.data_ptr(), out.second.data_ptr(), &desc,
                       st) != CL_OK)
        return c10::nullopt;
    return out;
}

bool cache_desc(const at::Tensor& k, const at::Tensor& v, const at::Tensor& pages,
                const at::Tensor& slots, cl_kvcache_desc* desc) {
    if (!k.is_cuda()) return false;
    const c10::DeviceIndex d = k.get_device();
    if (!rows_ok(k, 3, d) || !rows_ok(v, 3, d) || k.scalar_type() != v.scalar_type() ||
        k.sizes() != v.sizes() || !pages_ok(pages, k.size(2), d, &desc->bits, &desc->page_size) ||
        pages.size(1) != k.size(1) || !plain_ok(slots, 1, at::kLong, d) ||
        slots.size(0) != k.size(0))
        return false;
    desc->tokens = k.size(0);
    desc->num_pages = pages.size(0);
    desc->k_token = k.stride(0), desc->k_head = k.stride(1);
    desc->v_token = v.stride(0), desc->v_head = v.stride(1);
    desc->kv_heads = static_cast<int32_t>(k.size(1));
    desc->head_dim = static_cast<int32_t>(k.size(2));
    desc->dtype = type16(k);
    return true;
}

bool kvcache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& pages,
                   const at::Tensor& slots) {
    cl_kvcache_desc desc{};
    if (!cache_desc(k, v, pages, slots, &desc)) return false;
    c10::cuda::OptionalCUDAGuard guard;
    void* st = begin(k.get_device(), &guard);
    return cl_kvcache_write(k.data_ptr(), v.data_ptr(), static_cast<uint8_t*>(pages.data_ptr()),
                            slots.data_ptr<int64_t>(), &desc, st) == CL_OK;
}

c10::optional<Pair> kvcache_read(const at::Tensor& pages, const at::Tensor& slots,
                                 int64_t head_dim, bool bf16) {
    if (!pages.is_cuda() || pages.dim() != 4 || slots.dim() != 1 || head_dim <= 0 ||
        head_dim > 256)
        return c10::nullopt;
    const at::ScalarType type = bf16 ? at::kBFloat16 : at::kHalf;
    const c10::DeviceIndex d = pages.get_device();
    c10::cuda::OptionalCUDAGuard guard;
    void* st = begin(d, &guard);
    const std::array<int64_t, 3> shape = {slots.size(0), pages.size(1), head_dim};
    Pair out = empty_two(shape, type, shape, type, d);
    cl_kvcache_desc desc{};
    if (!cache_desc(out.first, out.second, pages, slots, &desc)) return c10::nullopt;
    if (cl_kvcache_read(static_cast<const uint8_t*>(pages.data_ptr()), slots.data_ptr<int64_t>(),
                        out.first.data_ptr(), out.second.data_ptr(), &desc, st) != CL_OK)
        return c10::nullopt;
    return out;
}

// out, or (out, lse); None when not taken.
py::object kvattention(const at::Tensor& q, const at::Tensor& pages, const at::Tensor& table,
                       const at::Tensor& lengths, const c10::optional<at::Tensor>& prefix,
                       int64_t prefix_length, double scale, bool default_scale, int64_t window,
                       const at::Tensor& workspace, bool return_lse) {
    if (!q.is_cuda() || (q.dim() != 3 && q.dim() != 4)) return py::none();
    const c10::DeviceIndex d = q.get_device();
    const int last = static_cast<int>(q.dim()) - 1;
    const int64_t B = q.size(0), new_tokens = last == 3 ? q.size(1) : 1, H = q.size(last - 1),
                  D = q.size(last);
    cl_kvattention_desc desc{};
    if (!rows_ok(q, last + 1, d) || !pages_ok(pages, D, d, &desc.bits, &desc.page_size) ||
        new_tokens <= 0 || new_tokens > (1 << 20) || B > 4096 || H <= 0 || H > (1 << 20) ||
        H % pages.size(1) != 0 || !plain_ok(lengths, 1, at::kInt, d) || lengths.size(0) != B ||
        table.dim() != 2 || table.size(0) != B || table.scalar_type() != at::kInt ||
        (table.size(1) > 1 && table.stride(1) != 1) || !on(table, d) || window < 0 ||
        window > INT32_MAX || table.size(1) > INT32_MAX ||
        !plain_ok(workspace, 1, at::kByte, d))
        return py::none();
    static const size_t need = [] {
        size_t n = 0;
        cl_kvattention_workspace(&n);
        return n;
    }();
    if (static_cast<size_t>(workspace.numel()) < need) return py::none();
    const bool shared = prefix_length > 0;
    if (shared && (!prefix.has_value() || !plain_ok(*prefix, 1, at::kInt, d) || window != 0 ||
                   prefix_length > prefix->size(0) * desc.page_size || prefix_length > INT32_MAX))
        return py::none();
    desc.num_pages = pages.size(0);
    desc.table_stride = table.stride(0);
    desc.q_batch = q.stride(0);
    desc.q_new = last == 3 ? q.stride(1) : 0;
    desc.q_head = q.stride(last - 1);
    desc.batch = static_cast<int32_t>(B);
    desc.new_tokens = static_cast<int32_t>(new_tokens);
    desc.q_heads = static_cast<int32_t>(H);
    desc.kv_heads = static_cast<int32_t>(pages.size(1));
    desc.head_dim = static_cast<int32_t>(D);
    desc.max_pages = static_cast<int32_t>(table.size(1));
    desc.window = static_cast<int32_t>(window);
    desc.dtype = type16(q);
    desc.scale = static_cast<float>(default_scale ? 1.0 / std::sqrt(static_cast<double>(D)) : scale);
    c10::cuda::OptionalCUDAGuard guard;
    void* st = begin(d, &guard);
    at::Tensor scratch;
    Pair result = return_lse ? empty_two(q.sizes(), q.scalar_type(), q.sizes().slice(0, last),
                                         at::kFloat, d)
                             : Pair(empty(q.sizes(), q.scalar_type(), d), at::Tensor());
    if (shared) {
        desc.prefix_length = static_cast<int32_t>(prefix_length);
        desc.prefix_page_count = static_cast<int32_t>(prefix->size(0));
        size_t floats = 0;
        if (cl_kvattention_prefix_floats(&desc, &floats) != CL_OK) return py::none();
        scratch = empty({static_cast<int64_t>(floats)}, at::kFloat, d);
    }
    if (cl_kvattention(q.data_ptr(), static_cast<const uint8_t*>(pages.data_ptr()),
                       table.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(),
                       shared ? prefix->data_ptr<int32_t>() : nullptr, result.first.data_ptr(),
                       return_lse ? result.second.data_ptr<float>() : nullptr,
                       shared ? scratch.data_ptr<float>() : nullptr, workspace.data_ptr(), &desc,
                       st) != CL_OK)
        return py::none();
    if (return_lse) return py::cast(result);
    return py::cast(result.first);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("qknorm_rope", &qknorm_rope, "norm and rotation of q and k (None when not taken)");
    m.def("kvcache_write", &kvcache_write, "quantise into the cache (False when not taken)");
    m.def("kvcache_read", &kvcache_read, "read the cache back (None when not taken)");
    m.def("kvattention", &kvattention, "attention over the cache (None when not taken)");
    m.attr("NOT_FAST") = kNotFast;
    m.def("forward_into", &forward_into, "checked GEMV into `out` (0 on success)");
    m.def("forward", &forward, "checked GEMV into a new tensor (None when not taken)");
}
