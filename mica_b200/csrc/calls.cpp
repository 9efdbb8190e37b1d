// calls.cpp -- the Python calls of the paged-cache and log-probability entry points: argument checks,
// outputs from torch's allocator, launch on the tensor's device and that device's current stream.
//
// A step of a few tokens takes the device less time than ctypes and Python-side checks take the host
// (append of 8 rows: 8 us against 21), so these calls are compiled. The library's entry points are
// handed over by address (bind), so both bindings use the same loaded library.
//
// Errors: ValueError for arguments that fit no call, RuntimeError for what the kernels do not serve,
// NativeError (raised by mica_b200._native.check) when an entry point returns a status.
#include <torch/extension.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAGuard.h>

#include <limits>
#include <sstream>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../include/mica_w8a8.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

decltype(&mica_cache_append) f_append = nullptr;
decltype(&mica_cache_attention) f_attention = nullptr;
decltype(&mica_cache_attention_workspace_bytes) f_attention_bytes = nullptr;
decltype(&mica_cache_copy) f_copy = nullptr;
decltype(&mica_cache_keep) f_keep = nullptr;
decltype(&mica_token_logprobs) f_logprobs = nullptr;
PyObject* g_check = nullptr;        // _native.check(name, rc)
PyObject* g_served = nullptr;       // (device index) -> bool, asked once a device
std::vector<signed char> g_device;  // -1 unknown

void bind(const std::unordered_map<std::string, uintptr_t>& at, py::object check, py::object served) {
    f_append = reinterpret_cast<decltype(f_append)>(at.at("mica_cache_append"));
    f_attention = reinterpret_cast<decltype(f_attention)>(at.at("mica_cache_attention"));
    f_attention_bytes = reinterpret_cast<decltype(f_attention_bytes)>(at.at("mica_cache_attention_workspace_bytes"));
    f_copy = reinterpret_cast<decltype(f_copy)>(at.at("mica_cache_copy"));
    f_keep = reinterpret_cast<decltype(f_keep)>(at.at("mica_cache_keep"));
    f_logprobs = reinterpret_cast<decltype(f_logprobs)>(at.at("mica_token_logprobs"));
    g_check = check.release().ptr();
    g_served = served.release().ptr();
}

template <typename... A>
[[noreturn]] void value(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    PyErr_SetString(PyExc_ValueError, s.str().c_str());
    throw py::error_already_set();
}
template <typename... A>
[[noreturn]] void runtime(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    throw std::runtime_error(s.str());
}
void status(const char* name, int rc) {
    if (rc) py::reinterpret_borrow<py::object>(g_check)(name, rc);
}

// All tensors on one served CUDA device.
void cuda(const char* name, const Tensor& t, std::initializer_list<const Tensor*> rest) {
    if (!t.is_cuda()) runtime(name, ": CUDA tensors only (this library has no CPU path)");
    for (const Tensor* r : rest)
        if (r && r->device() != t.device()) runtime(name, ": tensors on ", t.device().str(), " and ", r->device().str());
    const size_t i = static_cast<size_t>(t.get_device());
    if (i >= g_device.size()) g_device.resize(i + 1, -1);
    if (g_device[i] < 0) g_device[i] = py::reinterpret_borrow<py::object>(g_served)(i).cast<bool>() ? 1 : 0;
    if (!g_device[i]) runtime(name, ": ", t.device().str(), " is not a B200 (sm_100)");
}
// Neither gradients nor forward-mode tangents pass through these calls, and what they write is no leaf of a graph.
void no_grad(const char* name, std::initializer_list<const Tensor*> ts) {
    const bool grad = at::GradMode::is_enabled();
    for (const Tensor* t : ts) {
        if (grad && t->requires_grad()) runtime(name, ": no backward pass (call it under torch.no_grad())");
        if (t->_fw_grad(0).defined()) runtime(name, ": no forward-mode derivative");
    }
}
const Tensor* ptr(const OptTensor& t) { return t.has_value() ? &*t : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

struct Step {
    Tensor table, base, cu;     // rows of the table any distance apart; copies, made in the call, of what a kernel cannot read
    int B, P;
    long ld;
    Step(const char* name, const Tensor& t, const Tensor& b, const Tensor& c) : table(t), base(b), cu(c) {
        if (t.dim() != 2 || b.dim() != 1 || c.dim() != 1 || t.size(0) != b.size(0) || c.size(0) != b.size(0) + 1 ||
            t.size(1) < 1 || t.scalar_type() != at::kInt || b.scalar_type() != at::kInt || c.scalar_type() != at::kInt)
            value(name, ": table ", t.sizes(), ", base ", b.sizes(), ", cu ", c.sizes(), " (int32)");
        if (t.size(0) > std::numeric_limits<int>::max() || t.size(1) > std::numeric_limits<int>::max())
            value(name, ": table ", t.sizes());
        B = static_cast<int>(t.size(0));
        P = static_cast<int>(t.size(1));
    }
    void read() {               // on the call's device and stream
        if ((P > 1 && table.stride(1) != 1) || (B > 1 && table.stride(0) < P)) table = table.contiguous();
        base = base.contiguous();
        cu = cu.contiguous();
        ld = B > 1 ? table.stride(0) : P;
    }
};

struct Pages {
    int pages, kv, page, d;
    long stride;
    Pages(const char* name, const Tensor& k, const Tensor& v) {
        if (k.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides())
            value(name, ": K pages ", k.sizes(), " and V pages ", v.sizes());
        if (k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16)
            runtime(name, ": pages of ", k.scalar_type(), " are not served (bf16)");
        const int64_t n = k.size(0), h = k.size(1), p = k.size(2), c = k.size(3);
        if ((p != 16 && p != 32 && p != 64 && p != 128) || (c != 64 && c != 128) || k.stride(1) != p * c ||
            k.stride(2) != c || k.stride(3) != 1 || h < 1 || n < 1 || k.stride(0) < h * p * c ||
            n > std::numeric_limits<int>::max() || h > 4096)
            value(name, ": pages ", k.sizes(), " with strides ", k.strides(),
                  " (a page is [KV, page, D] contiguous, page 16, 32, 64 or 128, D 64 or 128)");
        pages = static_cast<int>(n); kv = static_cast<int>(h); page = static_cast<int>(p); d = static_cast<int>(c);
        stride = k.stride(0);
    }
};

// A matrix whose rows a kernel can read: unit columns, rows apart, 16-byte aligned (a copy otherwise).
Tensor rows16(const Tensor& t) {
    const bool fine = (t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0)) &&
                      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}
long row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void int_rows(const char* name, const Tensor& t) {
    if (t.size(0) > std::numeric_limits<int>::max()) value(name, ": ", t.size(0), " rows");
}

Tensor append(const Tensor& qkv_, const Tensor& q_w, const Tensor& k_w, const Tensor& cos, const Tensor& sin,
              const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& base, const Tensor& cu, int64_t heads,
              const OptTensor& pos_, double eps) {
    const char* name = "append";
    const Pages pg(name, k, v);
    Step st(name, table, base, cu);
    if (qkv_.dim() != 2 || heads < 1 || heads > 4096 || qkv_.size(1) != (heads + 2 * pg.kv) * pg.d || qkv_.stride(1) != 1)
        value(name, ": qkv ", qkv_.sizes(), " for ", heads, " + 2 x ", pg.kv, " heads of ", pg.d);
    if (q_w.dim() != 1 || q_w.size(0) != pg.d || k_w.sizes() != q_w.sizes() || cos.dim() != 2 || cos.sizes() != sin.sizes() ||
        cos.size(1) != pg.d)
        value(name, ": norms ", q_w.sizes(), ", ", k_w.sizes(), ", tables ", cos.sizes(), ", ", sin.sizes(), " for heads of ", pg.d);
    for (const Tensor* t : {&qkv_, &q_w, &k_w, &cos, &sin})
        if (t->scalar_type() != at::kBFloat16) runtime(name, ": bf16 tensors only");
    const int64_t n = qkv_.size(0);
    int_rows(name, qkv_);
    if (pos_ && (pos_->scalar_type() != at::kLong || pos_->dim() != 1 || pos_->size(0) != n))
        value(name, ": pos is int64 [", n, "], not ", pos_->scalar_type(), " ", pos_->sizes());
    if (!cos.is_contiguous() || !sin.is_contiguous() || cos.size(0) < 1) value(name, ": cos and sin are contiguous [positions, D]");
    cuda(name, qkv_, {&q_w, &k_w, &cos, &sin, &k, &v, &table, &base, &cu, ptr(pos_)});
    no_grad(name, {&qkv_, &q_w, &k_w, &k, &v});
    const c10::cuda::CUDAGuard guard(qkv_.device());
    st.read();
    if (n == 0 || st.B == 0) return at::zeros({n, heads * pg.d}, qkv_.options());      // padding rows alone
    const Tensor qkv = rows16(qkv_), qw = rows16(q_w.contiguous().unsqueeze(0)), kw = rows16(k_w.contiguous().unsqueeze(0));
    const Tensor pos = pos_ ? pos_->contiguous() : Tensor();
    Tensor q = at::empty({n, heads * pg.d}, qkv_.options());
    status("mica_cache_append",
           f_append(qkv.data_ptr(), row_stride(qkv), qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.size(0),
                    pos_ ? pos.data_ptr<int64_t>() : nullptr, q.data_ptr(), heads * pg.d, k.data_ptr(), v.data_ptr(), pg.stride,
                    pg.pages, pg.page, st.table.data_ptr<int>(), st.ld, st.P, st.base.data_ptr<int>(), st.cu.data_ptr<int>(), st.B,
                    static_cast<int>(n), static_cast<int>(heads), pg.kv, pg.d, static_cast<float>(eps), stream_of(qkv_)));
    return q;
}

Tensor attention(const Tensor& q_, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& base,
                 const Tensor& cu, const OptTensor& mask, int64_t heads, std::optional<double> scale_,
                 std::optional<int64_t> max_new) {
    const char* name = "attention";
    const Pages pg(name, k, v);
    Step st(name, table, base, cu);
    if (q_.dim() != 2 || heads < 1 || heads > 4096 || heads % pg.kv || heads / pg.kv > 128 || q_.size(1) != heads * pg.d ||
        q_.stride(1) != 1)
        value(name, ": q ", q_.sizes(), " for ", heads, " heads of ", pg.d, " over ", pg.kv, " K/V heads");
    if (q_.scalar_type() != at::kBFloat16) runtime(name, ": ", q_.scalar_type(), " is not served (bf16)");
    const int64_t n = q_.size(0);
    int_rows(name, q_);
    if (mask && (mask->dim() != 2 || mask->scalar_type() != at::kLong || mask->size(0) != n || mask->size(1) < 1 ||
                 mask->size(1) > (1 << 26)))
        value(name, ": mask ", mask->scalar_type(), " ", mask->sizes(), " for ", n, " rows (int64 [rows, words])");
    const double scale = scale_ ? *scale_ : 1.0 / std::sqrt(static_cast<double>(pg.d));
    if (!(scale > 0.0 && scale <= std::numeric_limits<float>::max())) value(name, ": scale ", scale);
    cuda(name, q_, {&k, &v, &table, &base, &cu, ptr(mask)});
    no_grad(name, {&q_, &k, &v});
    const c10::cuda::CUDAGuard guard(q_.device());
    st.read();
    if (n == 0 || st.B == 0) return at::zeros({n, heads * pg.d}, q_.options());
    const Tensor q = rows16(q_);
    Tensor out = at::empty({n, heads * pg.d}, q_.options());
    const int most = static_cast<int>(max_new ? std::min(*max_new, n) : n);
    const size_t need = f_attention_bytes(static_cast<int>(n), most, static_cast<int>(heads), pg.kv, pg.d);
    const Tensor ws = at::empty({static_cast<int64_t>(need)}, q_.options().dtype(at::kByte));
    const int words = mask ? static_cast<int>(mask->size(1)) : 0;
    const Tensor bits = !mask ? Tensor() : (words > 1 && mask->stride(1) != 1) || (n > 1 && mask->stride(0) < words) ? mask->contiguous() : *mask;
    status("mica_cache_attention",
           f_attention(q.data_ptr(), row_stride(q), k.data_ptr(), v.data_ptr(), pg.stride, pg.pages, pg.page,
                       st.table.data_ptr<int>(), st.ld, st.P, st.base.data_ptr<int>(), st.cu.data_ptr<int>(),
                       mask ? bits.data_ptr<int64_t>() : nullptr, mask && n > 1 ? bits.stride(0) : words, words, st.B, static_cast<int>(n), most,
                       static_cast<int>(heads), pg.kv, pg.d, static_cast<float>(scale), out.data_ptr(), heads * pg.d,
                       ws.data_ptr(), need, stream_of(q_)));
    return out;
}

long page_bytes(const char* name, const Tensor& pool) {
    const long es = static_cast<long>(pool.element_size());
    long n = 1;
    bool inner = pool.dim() >= 2 && pool.size(0) >= 1;
    for (int64_t i = pool.dim() - 1; inner && i > 0; --i) {
        inner = pool.size(i) == 1 || pool.stride(i) == n;
        n *= pool.size(i);
    }
    if (!inner || n == 0 || (pool.size(0) > 1 && pool.stride(0) < n) || reinterpret_cast<uintptr_t>(pool.data_ptr()) % 16 ||
        pool.stride(0) * es % 16 || n * es % 16 || pool.size(0) > std::numeric_limits<int>::max())
        value(name, ": pool ", pool.sizes(), " with strides ", pool.strides(), " (each page contiguous, whole 16-byte pieces)");
    return n * es;
}

void copy_pages(const Tensor& pool, const std::vector<int64_t>& src, const std::vector<int64_t>& dst) {
    const char* name = "copy_pages";
    const long bytes = page_bytes(name, pool);
    if (src.size() != dst.size()) value(name, ": ", src.size(), " pages onto ", dst.size());
    const int64_t pages = pool.size(0);
    std::vector<int> s, d;
    s.reserve(src.size());
    d.reserve(src.size());
    std::vector<bool> written(static_cast<size_t>(pages));
    for (size_t i = 0; i < src.size(); ++i) {
        if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages) value(name, ": a page outside the pool of ", pages);
        if (written[dst[i]]) value(name, ": page ", dst[i], " is written twice");
        written[dst[i]] = true;
        s.push_back(static_cast<int>(src[i]));
        d.push_back(static_cast<int>(dst[i]));
    }
    for (int64_t i : src)
        if (written[i]) value(name, ": page ", i, " is read and written");
    cuda(name, pool, {});
    no_grad(name, {&pool});
    if (s.empty()) return;
    const c10::cuda::CUDAGuard guard(pool.device());
    const long stride = pages > 1 ? pool.stride(0) * static_cast<long>(pool.element_size()) : bytes;
    status("mica_cache_copy", f_copy(pool.data_ptr(), stride, bytes, static_cast<int>(pages), s.data(), d.data(),
                                     static_cast<int>(s.size()), stream_of(pool)));
}

Tensor keep_tokens(const Tensor& pool, const Tensor& table, const Tensor& base, const Tensor& cu, const Tensor& keep_,
                   const Tensor& n_keep_) {
    const char* name = "keep_tokens";
    const auto one_of = [](int64_t x, std::initializer_list<int64_t> l) { return std::find(l.begin(), l.end(), x) != l.end(); };
    if (pool.dim() != 6 || pool.size(2) != 2 || pool.scalar_type() != at::kBFloat16 || !one_of(pool.size(4), {16, 32, 64, 128}) ||
        !one_of(pool.size(5), {64, 128}))
        value(name, ": pool ", pool.scalar_type(), " ", pool.sizes());
    const long bytes = page_bytes(name, pool);
    Step st(name, table, base, cu);
    if (keep_.dim() != 2 || keep_.size(0) != st.B || n_keep_.dim() != 1 || n_keep_.size(0) != st.B ||
        keep_.scalar_type() != at::kInt || n_keep_.scalar_type() != at::kInt || keep_.size(1) > std::numeric_limits<int>::max())
        value(name, ": keep ", keep_.scalar_type(), " ", keep_.sizes(), ", n_keep ", n_keep_.scalar_type(), " ", n_keep_.sizes(),
              " for ", st.B, " sequences (int32)");
    cuda(name, pool, {&table, &base, &cu, &keep_, &n_keep_});
    no_grad(name, {&pool});
    const c10::cuda::CUDAGuard guard(pool.device());
    st.read();
    if (st.B == 0 || keep_.size(1) == 0) return st.base.clone();
    const Tensor keep = keep_.contiguous(), n_keep = n_keep_.contiguous();
    Tensor out = at::empty_like(st.base);
    const int most = static_cast<int>(keep.size(1));
    const long stride = pool.size(0) > 1 ? pool.stride(0) * 2 : bytes;
    status("mica_cache_keep",
           f_keep(pool.data_ptr(), stride, static_cast<int>(pool.size(1) * 2 * pool.size(3)), static_cast<int>(pool.size(0)),
                  static_cast<int>(pool.size(4)), static_cast<int>(pool.size(5)), st.table.data_ptr<int>(), st.ld, st.P,
                  st.base.data_ptr<int>(), st.cu.data_ptr<int>(), st.B, keep.data_ptr<int>(), most, n_keep.data_ptr<int>(), most,
                  out.data_ptr<int>(), stream_of(pool)));
    return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& z_, const Tensor& ids_, int64_t top) {
    const char* name = "token_logprobs";
    if (z_.dim() != 2 || (ids_.dim() != 1 && ids_.dim() != 2) || ids_.size(0) != z_.size(0))
        value(name, ": logits ", z_.sizes(), " with ids ", ids_.sizes());
    if (ids_.scalar_type() != at::kLong) value(name, ": ids are int64, not ", ids_.scalar_type());
    const int64_t n = z_.size(0), v = z_.size(1);
    if (v < 1 || v > (1 << 30) || n > (1 << 30) || (ids_.dim() == 2 && ids_.size(1) > (1 << 30))) value(name, ": logits ", z_.sizes());
    if (top < 0 || top > 32 || top > v) value(name, ": top ", top, " of ", v, " tokens (at most 32)");
    cuda(name, z_, {&ids_});
    const int code = z_.scalar_type() == at::kBFloat16 ? MICA_DT_BF16 : z_.scalar_type() == at::kHalf ? MICA_DT_FP16
                     : z_.scalar_type() == at::kFloat ? MICA_DT_FP32 : -1;
    if (code < 0) runtime(name, ": ", z_.scalar_type(), " is not served (bf16, fp16 or fp32)");
    no_grad(name, {&z_});
    const c10::cuda::CUDAGuard guard(z_.device());
    const Tensor z = (v > 1 && z_.stride(1) != 1) || (n > 1 && z_.stride(0) < v) ? z_.contiguous() : z_;
    Tensor ids = ids_.dim() == 1 ? ids_.unsqueeze(1) : ids_;
    const int64_t m = ids.size(1);
    if ((m > 1 && ids.stride(1) != 1) || (n > 1 && ids.stride(0) < m)) ids = ids.contiguous();
    const auto f32 = z_.options().dtype(at::kFloat);
    Tensor lp = at::empty(ids_.sizes(), f32), ent = at::empty({n}, f32), top_lp = at::empty({n, top}, f32);
    Tensor top_id = at::empty({n, top}, z_.options().dtype(at::kLong));
    if (n > 0)
        status("mica_token_logprobs",
               f_logprobs(z.data_ptr(), code, n > 1 ? z.stride(0) : v, static_cast<int>(n), static_cast<int>(v),
                          m ? ids.data_ptr<int64_t>() : nullptr, n > 1 ? ids.stride(0) : m, static_cast<int>(m),
                          static_cast<int>(top), m ? lp.data_ptr<float>() : nullptr, ent.data_ptr<float>(),
                          top ? top_lp.data_ptr<float>() : nullptr, top ? top_id.data_ptr<int64_t>() : nullptr, stream_of(z_)));
    return {lp, ent, top_lp, top_id};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("bind", &bind);
    m.def("append", &append);
    m.def("attention", &attention);
    m.def("copy_pages", &copy_pages);
    m.def("keep_tokens", &keep_tokens);
    m.def("token_logprobs", &token_logprobs);
}
