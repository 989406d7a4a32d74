// rq_torch.cpp -- the paged serving operators of include/rq.h on torch tensors
// (module rustyllm_b200._rqtorch): the checks of arguments, the allocation of
// outputs and workspaces, and the current stream, in C++.  Single-token calls
// take a few microseconds on the GPU; the same in Python over ctypes cost 10 to
// 14 us of host time a call.

#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <string>

#include "../../include/rq.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

[[noreturn]] void raise(int code, const std::string& msg) {
    const py::object err = py::module_::import("rustyllm_b200._lib").attr("RqError");
    const py::object e = err(code, msg);
    PyErr_SetObject(err.ptr(), e.ptr());
    throw py::error_already_set();
}
[[noreturn]] void refuse(const std::string& msg) { raise(RQ_ERR_INVALID, msg); }

void check(int rc) {
    if (rc == RQ_OK) return;
    char buf[1024];
    rq_last_error(buf, sizeof buf);
    raise(rc, buf);
}

std::string cuda(int dev) { return "cuda:" + std::to_string(dev); }
bool on(const Tensor& t, int dev) { return t.is_cuda() && t.device().index() == dev; }

int dtype_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
    case at::kFloat: return RQ_F32;
    case at::kHalf: return RQ_F16;
    case at::kBFloat16: return RQ_BF16;
    default: raise(RQ_ERR_UNSUPPORTED, std::string(name) + ": " + c10::toString(t.scalar_type()) + " (float32, float16 or bfloat16)");
    }
}

// a contiguous int32 tensor (of n values where n >= 0) on the device
int32_t* ints(const Tensor& t, const char* name, int dev, int64_t n = -1) {
    if (!on(t, dev) || t.scalar_type() != at::kInt || !t.is_contiguous() || (n >= 0 && (t.dim() != 1 || t.size(0) != n)))
        refuse(std::string(name) + ": a contiguous int32 tensor" + (n >= 0 ? " of " + std::to_string(n) + " values" : "") + " on " +
               cuda(dev) + " is wanted");
    return t.data_ptr<int32_t>();
}
// [tokens, heads, dim] on the device with contiguous elements
void rows(const Tensor& t, const char* name, int64_t heads, int64_t dim, int dev) {
    if (!on(t, dev) || t.dim() != 3 || t.size(1) != heads || t.size(2) != dim || (dim != 1 && t.stride(2) != 1))
        refuse(std::string(name) + ": [tokens, " + std::to_string(heads) + ", " + std::to_string(dim) + "] on " + cuda(dev) +
               " with contiguous elements is wanted");
}
// a like-typed output of the same shape
void output(const Tensor& t, const Tensor& like, const char* name, int dev) {
    rows(t, name, like.size(1), like.size(2), dev);
    if (t.scalar_type() != like.scalar_type() || t.size(0) != like.size(0))
        refuse(std::string(name) + ": the shape and type of its input are wanted");
}
int table(const Tensor& t, int64_t batch, const char* name) {
    if (!t.is_cuda() || t.scalar_type() != at::kInt || t.dim() != 2 || (batch >= 0 && t.size(0) != batch) ||
        (t.size(1) > 1 && t.stride(1) != 1))
        refuse(std::string(name) + ": a CUDA int32 [batch, width] with contiguous rows is wanted");
    return t.device().index();
}
int small(int64_t n, const char* name) {
    if (n != (int)n) refuse(std::string(name) + " " + std::to_string(n) + " is out of range");
    return (int)n;
}
Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor new_ints(at::IntArrayRef shape, int dev) {
    return at::empty(shape, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)dev));
}
void* stream_of(int dev) { return at::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
void pair(int64_t (&s)[2], const Tensor& t) {
    s[0] = t.stride(0);
    s[1] = t.stride(1);
}

// ------------------------------------------------------------------ cache

struct Cache {
    rq_kv4* handle;  // NULL once closed: the entries refuse it
    int64_t heads, dim;
    int dev;
};

void append(const Cache& c, const Tensor& k, const Tensor& v, const Tensor& slots) {
    rows(k, "k", c.heads, c.dim, c.dev);
    rows(v, "v", c.heads, c.dim, c.dev);
    if (k.scalar_type() != v.scalar_type() || k.size(0) != v.size(0)) refuse("append: k and v differ in type or length");
    const int32_t* s = ints(slots, "slots", c.dev, k.size(0));
    int64_t ks[2], vs[2];
    pair(ks, k);
    pair(vs, v);
    check(rq_kv4_append(c.handle, dtype_of(k, "k"), k.data_ptr(), ks, v.data_ptr(), vs, s, k.size(0), stream_of(c.dev)));
}

py::tuple read(const Cache& c, const Tensor& slots, at::ScalarType type) {
    const int32_t* s = ints(slots, "slots", c.dev, slots.numel());
    const Tensor kv = at::empty({2, slots.numel(), c.heads, c.dim}, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)c.dev));
    const int dt = dtype_of(kv, "dtype");
    Tensor k = kv.select(0, 0), v = kv.select(0, 1);
    check(rq_kv4_read(c.handle, s, slots.numel(), dt, k.data_ptr(), v.data_ptr(), stream_of(c.dev)));
    return py::make_tuple(std::move(k), std::move(v));
}

Tensor attention(const Cache& c, const Tensor& q, const Tensor& block_table, const Tensor& kv_lens, const OptTensor& cu_q,
                 const std::optional<int64_t>& max_q, double scale, int64_t window, const OptTensor& out, int64_t max_len) {
    if (q.dim() != 3) refuse("q: [tokens, heads, head_dim] is wanted");
    rows(q, "q", q.size(1), c.dim, c.dev);
    if (table(block_table, -1, "block_table") != c.dev) refuse("block_table: on " + cuda(c.dev) + " is wanted");
    const int64_t batch = block_table.size(0);
    rq_kv4_query a{};
    a.kv_lens = ints(kv_lens, "kv_lens", c.dev, batch);
    if (cu_q) a.cu_q = ints(*cu_q, "cu_q", c.dev, batch + 1);
    if (out) output(*out, q, "out", c.dev);
    a.dtype = dtype_of(q, "q");
    Tensor o = out ? *out : like(q);
    a.q = q.data_ptr();
    pair(a.q_stride, q);
    a.out = o.data_ptr();
    pair(a.out_stride, o);
    a.n_tokens = q.size(0);
    a.n_heads = q.size(1);
    a.batch = batch;
    a.max_q = max_q ? *max_q : cu_q ? std::max<int64_t>(q.size(0), 1) : 1;
    a.block_table = block_table.data_ptr<int32_t>();
    a.table_stride = block_table.stride(0);
    a.table_width = block_table.size(1);
    a.max_len = max_len;
    a.window = window;
    a.scale = (float)scale;
    size_t need = 0;
    check(rq_kv4_attention_workspace(c.handle, &a, &need));
    Tensor ws;  // of the current stream's (and a captured graph's own) pool
    if (need) {
        ws = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, (c10::DeviceIndex)c.dev));
        a.workspace = ws.data_ptr();
        a.workspace_bytes = need;
    }
    check(rq_kv4_attention(c.handle, &a, stream_of(c.dev)));
    return o;
}

// ------------------------------------------------------ norm and rotation

rq_qk_rope rope_args(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& cos, const Tensor& sin,
                     const OptTensor& qw, const OptTensor& kw, double eps, bool interleaved, OptTensor& q_out, OptTensor& k_out,
                     bool append) {
    if (!q.is_cuda() || q.dim() != 3 || k.dim() != 3 || q.scalar_type() != k.scalar_type() || q.size(0) != k.size(0))
        refuse("q, k: [tokens, heads, head_dim] of one type on one CUDA device are wanted");
    const int dev = q.device().index();
    const int64_t hd = q.size(2);
    rows(q, "q", q.size(1), hd, dev);
    rows(k, "k", k.size(1), hd, dev);
    rq_qk_rope a{};
    a.dtype = dtype_of(q, "q");
    if (q_out) output(*q_out, q, "q_out", dev);
    else q_out = like(q);
    if (k_out) output(*k_out, k, "k_out", dev);
    else if (!append) k_out = like(k);
    if (!on(cos, dev) || !on(sin, dev) || cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 ||
        cos.sizes() != sin.sizes() || !cos.is_contiguous() || !sin.is_contiguous())
        refuse("cos, sin: contiguous float32 [max_pos, rot_dim / 2] on " + cuda(dev) + " are wanted");
    for (const OptTensor* w : {&qw, &kw})
        if (*w && (!on(**w, dev) || (*w)->scalar_type() != at::kFloat || (*w)->dim() != 1 || (*w)->size(0) != hd || !(*w)->is_contiguous()))
            refuse("q_weight, k_weight: contiguous float32 [" + std::to_string(hd) + "] on " + cuda(dev) + " are wanted");
    a.positions = ints(positions, "positions", dev, q.size(0));
    a.n_tokens = q.size(0);
    a.n_heads = q.size(1);
    a.n_kv_heads = k.size(1);
    a.head_dim = hd;
    a.rot_dim = 2 * cos.size(1);
    a.interleaved = interleaved;
    a.q = q.data_ptr();
    pair(a.q_stride, q);
    a.q_out = q_out->data_ptr();
    pair(a.q_out_stride, *q_out);
    a.k = k.data_ptr();
    pair(a.k_stride, k);
    if (k_out) {
        a.k_out = k_out->data_ptr();
        pair(a.k_out_stride, *k_out);
    }
    a.q_weight = qw ? qw->data_ptr<float>() : nullptr;
    a.k_weight = kw ? kw->data_ptr<float>() : nullptr;
    a.eps = (float)eps;
    a.cos = cos.data_ptr<float>();
    a.sin = sin.data_ptr<float>();
    a.max_pos = cos.size(0);
    return a;
}

py::tuple qk_norm_rope(uintptr_t ctx, const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& cos,
                       const Tensor& sin, const OptTensor& qw, const OptTensor& kw, double eps, bool interleaved, OptTensor q_out,
                       OptTensor k_out) {
    const rq_qk_rope a = rope_args(q, k, positions, cos, sin, qw, kw, eps, interleaved, q_out, k_out, false);
    check(rq_qk_norm_rope((rq_ctx*)ctx, &a, stream_of(q.device().index())));
    return py::make_tuple(*q_out, *k_out);
}

Tensor qk_norm_rope_append(const Cache& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions,
                           const Tensor& slots, const Tensor& cos, const Tensor& sin, const OptTensor& qw, const OptTensor& kw,
                           double eps, bool interleaved, OptTensor q_out) {
    rows(k, "k", c.heads, c.dim, c.dev);
    rows(v, "v", c.heads, c.dim, c.dev);
    if (v.scalar_type() != k.scalar_type() || v.size(0) != k.size(0)) refuse("v: the shape and type of k are wanted");
    OptTensor none;
    const rq_qk_rope a = rope_args(q, k, positions, cos, sin, qw, kw, eps, interleaved, q_out, none, true);
    const int32_t* s = ints(slots, "slots", c.dev, q.size(0));
    int64_t vs[2];
    pair(vs, v);
    check(rq_qk_norm_rope_append(c.handle, &a, v.data_ptr(), vs, s, stream_of(c.dev)));
    return *q_out;
}

// ------------------------------------------------------------------ pages

py::tuple pages_extend(uintptr_t ctx, const Tensor& ctx_lens, const Tensor& new_lens, const Tensor& tab, const Tensor& ring,
                       const Tensor& state, int64_t page_size, int64_t n_tokens, const OptTensor& state_out,
                       const OptTensor& kv_lens_out) {
    const int64_t batch = new_lens.numel();
    const int dev = table(tab, batch, "table");
    const int32_t* c = ints(ctx_lens, "ctx_lens", dev, batch);
    const int32_t* f = ints(new_lens, "new_lens", dev, batch);
    const int32_t* r = ints(ring, "ring", dev);
    const int32_t* st = ints(state, "free", dev, 3);
    if (n_tokens < 0) refuse("pages_extend: n_tokens " + std::to_string(n_tokens));
    // one allocation: state, lengths, offsets, positions, slots
    const Tensor buf = new_ints({4 + 2 * batch + 2 * n_tokens}, dev);
    Tensor so = state_out ? *state_out : buf.narrow(0, 0, 3), kv = kv_lens_out ? *kv_lens_out : buf.narrow(0, 3, batch);
    if (state_out) ints(so, "free_out", dev, 3);
    if (kv_lens_out) ints(kv, "kv_lens_out", dev, batch);
    int32_t* cu = buf.data_ptr<int32_t>() + 3 + batch;
    int32_t* pos = cu + batch + 1;
    check(rq_pages_extend((rq_ctx*)ctx, batch, small(page_size, "page_size"), c, f, tab.data_ptr<int32_t>(), tab.stride(0), tab.size(1), r,
                          ring.numel(), st, so.data_ptr<int32_t>(), kv.data_ptr<int32_t>(), cu, pos, pos + n_tokens, n_tokens,
                          stream_of(dev)));
    return py::make_tuple(std::move(so), std::move(kv), buf.narrow(0, 3 + batch, batch + 1),
                          buf.narrow(0, 4 + 2 * batch, n_tokens), buf.narrow(0, 4 + 2 * batch + n_tokens, n_tokens));
}

void pages_release(uintptr_t ctx, const Tensor& held, const Tensor& keep, const Tensor& tab, const Tensor& ring,
                   const Tensor& state, int64_t page_size) {
    const int64_t batch = held.numel();
    const int dev = table(tab, batch, "table");
    const int32_t* h = ints(held, "held_lens", dev, batch);
    const int32_t* k = ints(keep, "keep_lens", dev, batch);
    int32_t* r = ints(ring, "ring", dev);
    int32_t* st = ints(state, "free", dev, 3);
    check(rq_pages_release((rq_ctx*)ctx, batch, small(page_size, "page_size"), h, k, tab.data_ptr<int32_t>(), tab.stride(0), tab.size(1), r,
                           ring.numel(), st, stream_of(dev)));
}

// ----------------------------------------------------------- verification

py::tuple spec_verify(uintptr_t ctx, const Tensor& p, const Tensor& drafts, const Tensor& u, const Tensor& r, const OptTensor& q,
                      const OptTensor& n_drafts) {
    if (!p.is_cuda() || p.dim() != 3 || p.size(1) < 1 || (p.size(2) > 1 && p.stride(2) != 1))
        refuse("p: a CUDA tensor [batch, n + 1, vocab] with contiguous rows is wanted");
    const int64_t b = p.size(0), n = p.size(1) - 1, vocab = p.size(2);
    const int dev = p.device().index();
    const std::string bn = "[" + std::to_string(b) + ", " + std::to_string(n) + "]";
    if (q && (!on(*q, dev) || q->scalar_type() != p.scalar_type() || q->dim() != 3 || q->size(0) != b || q->size(1) != n ||
              q->size(2) != vocab || (n && vocab > 1 && q->stride(2) != 1)))
        refuse("q: [batch, n, vocab] of p's type with contiguous rows on " + cuda(dev) + " is wanted");
    const int32_t* d = ints(drafts, "drafts", dev);
    if (drafts.dim() != 2 || drafts.size(0) != b || drafts.size(1) != n) refuse("drafts: " + bn + " is wanted");
    if (!on(u, dev) || u.scalar_type() != at::kFloat || u.dim() != 2 || u.size(0) != b || u.size(1) != n || !u.is_contiguous())
        refuse("u: a contiguous float32 " + bn + " on " + cuda(dev) + " is wanted");
    if (!on(r, dev) || r.scalar_type() != at::kFloat || r.dim() != 1 || r.size(0) != b || !r.is_contiguous())
        refuse("r: a contiguous float32 [" + std::to_string(b) + "] on " + cuda(dev) + " is wanted");
    const int32_t* nd = n_drafts ? ints(*n_drafts, "n_drafts", dev, b) : nullptr;
    const int dt = dtype_of(p, "p");
    const Tensor tokens = new_ints({b, n + 1}, dev), accepted = new_ints({b}, dev);
    int64_t ps[2], qs[2] = {0, 0};
    pair(ps, p);
    if (q) pair(qs, *q);
    check(rq_spec_verify((rq_ctx*)ctx, dt, p.data_ptr(), ps, q ? q->data_ptr() : nullptr, qs, d, nd, u.data_ptr<float>(),
                         r.data_ptr<float>(), b, n, vocab, tokens.data_ptr<int32_t>(), accepted.data_ptr<int32_t>(),
                         stream_of(dev)));
    return py::make_tuple(tokens, accepted);
}

}  // namespace

PYBIND11_MODULE(_rqtorch, m) {
    py::class_<Cache>(m, "Cache").def(py::init([](uintptr_t handle, int64_t heads, int64_t dim, int dev) {
        return Cache{(rq_kv4*)handle, heads, dim, dev};
    })).def("close", [](Cache& c) { c.handle = nullptr; });
    m.def("append", &append);
    m.def("read", [](const Cache& c, const Tensor& slots, py::object dtype) {
        return read(c, slots, torch::python::detail::py_object_to_dtype(std::move(dtype)));
    });
    m.def("attention", &attention);
    m.def("qk_norm_rope", &qk_norm_rope);
    m.def("qk_norm_rope_append", &qk_norm_rope_append);
    m.def("pages_extend", &pages_extend);
    m.def("pages_release", &pages_release);
    m.def("spec_verify", &spec_verify);
}
