// The paged operators' calls from PyTorch tensors: argument checks, output and
// workspace allocation and the C call, in one native function each.  In Python
// those take 20 us, several times what the kernels of a small decode step do.
// The C functions are bound by address (bind()), so this file does not link
// against the library.  Errors are RuntimeErrors, as everywhere in ops.
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "hq4.h"

namespace {

decltype(&hq4_paged_append) c_append = nullptr;
decltype(&hq4_paged_attention) c_attention = nullptr;
decltype(&hq4_tree_attention) c_tree = nullptr;
decltype(&hq4_paged_attention_workspace_bytes) c_workspace = nullptr;
decltype(&hq4_sample_rows) c_sample = nullptr;
PyObject* check_fn = nullptr;  // _lib.check: raises for a return code

// A failed check: the message goes into a RuntimeError.
void say(std::string& s, const char* v) { s += v; }
void say(std::string& s, long long v) { s += std::to_string(v); }
void say(std::string& s, c10::Device v) { s += v.str(); }
void say(std::string& s, at::IntArrayRef v) {
    s += '[';
    for (size_t i = 0; i < v.size(); i++) {
        if (i) s += ", ";
        s += std::to_string(v[i]);
    }
    s += ']';
}
template <class... Args>
[[noreturn]] void refuse(const Args&... args) {
    std::string s;
    (say(s, args), ...);
    throw std::runtime_error(s);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(name, " must be a torch.Tensor");
    return THPVariable_Unpack(o);
}
// An optional tensor: undefined for None.
at::Tensor maybe(PyObject* o, const char* name) { return o == Py_None ? at::Tensor() : tensor(o, name); }

int type_code(at::ScalarType t) {
    return t == at::kFloat ? HQ4_F32 : t == at::kBFloat16 ? HQ4_BF16 : t == at::kHalf ? HQ4_F16 : -1;
}
const char* type_name(at::ScalarType t) { return c10::toString(t); }
template <class T>
T* ptr(const at::Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// Contiguous, on `dev`, of a type and, where given, a number of dimensions.
void need(const at::Tensor& t, const char* name, at::ScalarType type, c10::Device dev) {
    if (!t.is_cuda()) refuse(name, " must be a CUDA tensor (no CPU fallback)");
    if (t.device() != dev) refuse(name, " must be on ", dev, ", is on ", t.device());
    if (t.scalar_type() != type) refuse(name, " must be ", type_name(type), ", got ", type_name(t.scalar_type()));
    if (!t.is_contiguous()) refuse(name, " must be contiguous");
}
// [rows, heads, head_dim] whose rows may be apart (a view of a fused projection).
void need_rows(const at::Tensor& t, const char* name, int64_t heads, int64_t head_dim, const at::Tensor* like) {
    if (t.dim() != 3 || (heads >= 0 && t.size(1) != heads) || (head_dim >= 0 && t.size(2) != head_dim))
        refuse(name, " must be [rows, heads, head_dim], got ", t.sizes());
    if (!t.is_cuda()) refuse(name, " must be a CUDA tensor (no CPU fallback)");
    if (type_code(t.scalar_type()) < 0)
        refuse(name, " must be float32, bfloat16 or float16, got ", type_name(t.scalar_type()));
    if (t.stride(2) != 1 || (t.size(1) > 1 && t.stride(1) != t.size(2)))
        refuse(name, "'s heads must lie one after another within a row");
    if (like && (t.scalar_type() != like->scalar_type() || t.size(0) != like->size(0) || t.device() != like->device()))
        refuse(name, " must have q's rows, type and device");
}
// Elements from a row to the next (a lone row has none of its own).
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); }
int64_t page_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2) * t.size(3); }

int fit(int64_t v, const char* name) {
    if (v < 0 || v > 0x7fffffff) refuse(name, " is too large");
    return (int)v;
}

struct Caches {
    int n_pages, n_kv, page_size, head_dim, type;
    int64_t stride;
};
Caches need_caches(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
    const at::Tensor* both[2] = {&k, &v};
    const char* names[2] = {"k_cache", "v_cache"};
    for (int i = 0; i < 2; i++) {
        const at::Tensor& t = *both[i];
        if (t.dim() != 4 || !t.is_cuda() || t.device() != q.device())
            refuse(names[i], " must be a CUDA tensor [n_pages, n_kv, page_size, head_dim] on ", q.device());
        if ((t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kHalf) || t.scalar_type() != k.scalar_type())
            refuse("the caches must be both bfloat16 or both float16");
        if (t.stride(3) != 1 || t.stride(2) != t.size(3) || (t.size(1) > 1 && t.stride(1) != t.size(2) * t.size(3)))
            refuse(names[i], "'s pages must each be contiguous");
    }
    if (v.sizes() != k.sizes() || page_stride(v) != page_stride(k))
        refuse("k_cache and v_cache must have the same shape and strides");
    if (q.scalar_type() != at::kFloat && q.scalar_type() != k.scalar_type())
        refuse("activations must be float32 or the caches' ", type_name(k.scalar_type()), ", got ", type_name(q.scalar_type()));
    if (q.device().index() != c10::cuda::current_device())
        refuse("tensors on ", q.device(), ", current device ", (long long)c10::cuda::current_device());
    return {fit(k.size(0), "n_pages"), fit(k.size(1), "n_kv"), fit(k.size(2), "page_size"), fit(k.size(3), "head_dim"),
            type_code(k.scalar_type()), page_stride(k)};
}
int need_batch(const at::Tensor& q, const at::Tensor& pages, const at::Tensor& cu_rows, const at::Tensor& lens) {
    need(lens, "lens", at::kInt, q.device());
    need(cu_rows, "cu_rows", at::kInt, q.device());
    need(pages, "pages", at::kInt, q.device());
    if (lens.dim() != 1) refuse("lens must be [n_seqs], got ", lens.sizes());
    const int64_t n = lens.size(0);
    if (cu_rows.dim() != 1 || cu_rows.size(0) != n + 1) refuse("cu_rows must be [n_seqs + 1], got ", cu_rows.sizes());
    if (pages.dim() != 2 || pages.size(0) != n) refuse("pages must be [n_seqs, pages_per_seq], got ", pages.sizes());
    return fit(n, "n_seqs");
}
at::Tensor output(const at::Tensor& out, const at::Tensor& q) {
    if (!out.defined())
        return at::detail::empty_cuda(q.sizes(), q.scalar_type(), q.device(), std::nullopt);
    need(out, "out", q.scalar_type(), q.device());
    if (out.sizes() != q.sizes()) refuse("out must have q's shape");
    return out;
}
void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

struct PyError {};  // a Python error is set
void check(int rc, const char* what) {
    if (rc == 0) return;
    PyObject* r = PyObject_CallFunction(check_fn, "is", rc, what);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) refuse(what, " failed with ", (long long)rc);
    throw PyError{};
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PyError{};
    return v;
}
// C++ errors do not leave the module.
template <class F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const PyError&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}
bool count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, got %zd", want, n);
    return false;
}

// q, k, v, k_cache, v_cache, pages, cu_rows, lens, rope_cos, rope_sin, positions, q_norm, k_norm, eps, out
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 15)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
        const at::Tensor &kc = tensor(a[3], "k_cache"), &vc = tensor(a[4], "v_cache");
        const at::Tensor &pages = tensor(a[5], "pages"), &cu = tensor(a[6], "cu_rows"), &lens = tensor(a[7], "lens");
        const at::Tensor &cos = tensor(a[8], "rope_cos"), &sin = tensor(a[9], "rope_sin");
        const at::Tensor pos = maybe(a[10], "positions"), qn = maybe(a[11], "q_norm"), kn = maybe(a[12], "k_norm");
        const float eps = (float)number(a[13]);
        need_rows(q, "q", -1, kc.dim() == 4 ? kc.size(3) : -1, nullptr);
        const Caches c = need_caches(q, kc, vc);
        need_rows(k, "k", c.n_kv, c.head_dim, &q);
        need_rows(v, "v", c.n_kv, c.head_dim, &q);
        const int n_seqs = need_batch(q, pages, cu, lens);
        need(cos, "rope_cos", at::kFloat, q.device());
        need(sin, "rope_sin", at::kFloat, q.device());
        if (cos.dim() != 2 || cos.size(1) * 2 != c.head_dim || sin.sizes() != cos.sizes())
            refuse("rope_cos and rope_sin must be [max_pos, head_dim / 2]");
        const at::Tensor* norms[2] = {&qn, &kn};
        for (int i = 0; i < 2; i++)
            if (norms[i]->defined()) {
                need(*norms[i], i ? "k_norm" : "q_norm", at::kFloat, q.device());
                if (norms[i]->dim() != 1 || norms[i]->size(0) != c.head_dim) refuse(i ? "k_norm" : "q_norm", " must be [head_dim]");
            }
        if (pos.defined()) {
            need(pos, "positions", at::kInt, q.device());
            if (pos.dim() != 1 || pos.size(0) != q.size(0)) refuse("positions must be [rows]");
        }
        const at::Tensor out = output(maybe(a[14], "out"), q);
        if (q.size(0))
            check(c_append(q.data_ptr(), k.data_ptr(), v.data_ptr(), type_code(q.scalar_type()), fit(q.size(0), "rows"),
                           fit(q.size(1), "n_heads"), c.n_kv, c.head_dim, row_stride(q), row_stride(k), row_stride(v),
                           ptr<float>(qn), ptr<float>(kn), eps, ptr<int>(cu), ptr<int>(lens), n_seqs, ptr<int>(pos),
                           ptr<float>(cos), ptr<float>(sin), fit(cos.size(0), "max_pos"), ptr<int>(pages),
                           fit(pages.size(1), "pages_per_seq"), kc.data_ptr(), vc.data_ptr(), c.type, c.n_pages,
                           c.page_size, c.stride, out.data_ptr(), stream_of(q)),
                  "hq4_paged_append");
        if (a[14] != Py_None) return Py_NewRef(a[14]);
        return THPVariable_Wrap(out);
    });
}

int64_t workspace_bytes(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& pages) {
    const long long b = c_workspace(type_code(q.scalar_type()), fit(q.size(0), "rows"), fit(q.size(1), "n_heads"),
                                    fit(kc.size(1), "n_kv"), fit(q.size(2), "head_dim"), fit(pages.size(0), "n_seqs"),
                                    fit(pages.size(1), "pages_per_seq"), fit(kc.size(2), "page_size"));
    if (b < 0)
        refuse("hq4_paged_attention_workspace_bytes = ", b, " for q ", q.sizes(), ", cache ", kc.sizes(), ", pages ", pages.sizes());
    return b;
}

// q, k_cache, v_cache, pages, cu_rows, lens, tree_mask, scale, out, workspace
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 10)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache");
        const at::Tensor &pages = tensor(a[3], "pages"), &cu = tensor(a[4], "cu_rows"), &lens = tensor(a[5], "lens");
        const at::Tensor mask = maybe(a[6], "tree_mask");
        need_rows(q, "q", -1, kc.dim() == 4 ? kc.size(3) : -1, nullptr);
        const Caches c = need_caches(q, kc, vc);
        const int n_seqs = need_batch(q, pages, cu, lens);
        if (mask.defined()) {
            need(mask, "tree_mask", at::kInt, q.device());
            if (mask.dim() != 2 || mask.size(0) != q.size(0) || mask.size(1) < 1)
                refuse("tree_mask must be [rows, words], got ", mask.sizes());
        }
        const float scale = (float)(a[7] == Py_None ? 1.0 / std::sqrt((double)c.head_dim) : number(a[7]));
        const at::Tensor out = output(maybe(a[8], "out"), q);
        if (q.size(0)) {
            at::Tensor ws = maybe(a[9], "workspace");
            if (ws.defined()) need(ws, "workspace", at::kByte, q.device());
            else if (const int64_t b = workspace_bytes(q, kc, pages))
                ws = at::detail::empty_cuda({b}, at::kByte, q.device(), std::nullopt);
            void* wp = ws.defined() && ws.numel() ? ws.data_ptr() : nullptr;
            const long long wb = ws.defined() ? ws.numel() : 0;
            const int t = type_code(q.scalar_type()), rows = fit(q.size(0), "rows"), heads = fit(q.size(1), "n_heads");
            const int per = fit(pages.size(1), "pages_per_seq");
            if (mask.defined())
                check(c_tree(q.data_ptr(), t, rows, heads, c.n_kv, c.head_dim, row_stride(q), ptr<int>(cu), ptr<int>(lens),
                             n_seqs, ptr<int>(pages), per, kc.data_ptr(), vc.data_ptr(), c.type, c.n_pages, c.page_size,
                             c.stride, reinterpret_cast<uint32_t*>(ptr<int>(mask)), fit(mask.size(1), "words"), scale,
                             out.data_ptr(), wp, wb, stream_of(q)),
                      "hq4_tree_attention");
            else
                check(c_attention(q.data_ptr(), t, rows, heads, c.n_kv, c.head_dim, row_stride(q), ptr<int>(cu),
                                  ptr<int>(lens), n_seqs, ptr<int>(pages), per, kc.data_ptr(), vc.data_ptr(), c.type,
                                  c.n_pages, c.page_size, c.stride, scale, out.data_ptr(), wp, wb, stream_of(q)),
                      "hq4_paged_attention");
        }
        if (a[8] != Py_None) return Py_NewRef(a[8]);
        return THPVariable_Wrap(out);
    });
}

// q, k_cache, pages
PyObject* workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 3)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &pages = tensor(a[2], "pages");
        need_rows(q, "q", -1, kc.dim() == 4 ? kc.size(3) : -1, nullptr);
        if (kc.dim() != 4 || pages.dim() != 2) refuse("k_cache must be [n_pages, n_kv, page_size, head_dim], pages [n_seqs, pages_per_seq]");
        const int64_t b = q.size(0) ? workspace_bytes(q, kc, pages) : 0;
        return THPVariable_Wrap(at::detail::empty_cuda({b}, at::kByte, q.device(), std::nullopt));
    });
}

// logits, u, temperature, top_k, top_p, min_p, out, logprob
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 8)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0], "logits");
        const int want = PyObject_IsTrue(a[7]);
        if (want < 0) throw PyError{};
        if (x.dim() != 2 || !x.is_cuda() || type_code(x.scalar_type()) < 0)
            refuse("logits must be a CUDA float32, bfloat16 or float16 tensor [rows, vocab]");
        const int64_t rows = x.size(0), vocab = x.size(1);
        if (vocab > 1 && x.stride(1) != 1) refuse("logits' rows must each be contiguous");
        if (x.device().index() != c10::cuda::current_device())
            refuse("tensors on ", x.device(), ", current device ", (long long)c10::cuda::current_device());
        static const char* const names[6] = {"u", "temperature", "top_k", "top_p", "min_p", "out"};
        static const at::ScalarType types[6] = {at::kDouble, at::kFloat, at::kInt, at::kFloat, at::kFloat, at::kInt};
        at::Tensor t[6];
        for (int i = 0; i < 6; i++) {
            t[i] = i ? maybe(a[i + 1], names[i]) : tensor(a[1], names[0]);
            if (!t[i].defined()) continue;
            need(t[i], names[i], types[i], x.device());
            if (t[i].dim() != 1 || t[i].size(0) != rows) refuse(names[i], " must be [rows], got ", t[i].sizes());
        }
        const bool given = t[5].defined();
        if (!given) t[5] = at::detail::empty_cuda({rows}, at::kInt, x.device(), std::nullopt);
        at::Tensor lp;
        if (want) lp = at::detail::empty_cuda({rows}, at::kFloat, x.device(), std::nullopt);
        if (rows)
            check(c_sample(x.data_ptr(), type_code(x.scalar_type()), fit(rows, "rows"), fit(vocab, "vocab"),
                           rows > 1 ? x.stride(0) : vocab, ptr<float>(t[1]), ptr<int>(t[2]), ptr<float>(t[3]),
                           ptr<float>(t[4]), ptr<double>(t[0]), ptr<int>(t[5]), ptr<float>(lp), stream_of(x)),
                  "hq4_sample_rows");
        PyObject* tok = given ? Py_NewRef(a[6]) : THPVariable_Wrap(t[5]);
        if (!want) return tok;
        PyObject* l = tok ? THPVariable_Wrap(lp) : nullptr;
        PyObject* both = l ? PyTuple_Pack(2, tok, l) : nullptr;
        Py_XDECREF(tok);
        Py_XDECREF(l);
        return both;
    });
}

// bind(check, {name: address}): the library's functions.
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *fn, *table;
    if (!PyArg_ParseTuple(args, "OO!", &fn, &PyDict_Type, &table)) return nullptr;
    auto at = [&](const char* name) -> void* {
        PyObject* v = PyDict_GetItemString(table, name);
        if (!v) {
            PyErr_Format(PyExc_KeyError, "%s", name);
            return nullptr;
        }
        return PyLong_AsVoidPtr(v);
    };
    void* f[5] = {at("hq4_paged_append"), at("hq4_paged_attention"), at("hq4_tree_attention"),
                  at("hq4_paged_attention_workspace_bytes"), at("hq4_sample_rows")};
    if (PyErr_Occurred()) return nullptr;
    c_append = reinterpret_cast<decltype(c_append)>(f[0]);
    c_attention = reinterpret_cast<decltype(c_attention)>(f[1]);
    c_tree = reinterpret_cast<decltype(c_tree)>(f[2]);
    c_workspace = reinterpret_cast<decltype(c_workspace)>(f[3]);
    c_sample = reinterpret_cast<decltype(c_sample)>(f[4]);
    Py_INCREF(fn);
    Py_XSETREF(check_fn, fn);
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr}, {"paged_append", FAST(append)},
                         {"attend", FAST(attend)},              {"workspace", FAST(workspace)},
                         {"sample_rows", FAST(sample)},         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hq4_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hq4_torch() { return PyModule_Create(&module); }
