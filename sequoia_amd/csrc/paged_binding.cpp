// The paged operators' way from torch tensors to the C entries: checks, workspaces, stream, call.  A call of theirs is a few
// microseconds of device work, many times a step, and the same checks in Python with a call through ctypes cost more than the launch:
// one token's attention 8.9 us, 4.4 by this way; a short read 8.2 | 4.3; a verification, three launches, 15.0 | 11.3.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>

#include <limits>
#include <string>

#include "../../include/sequoia_hip.h"

namespace {

using at::ScalarType;
using at::Tensor;

// from bind(): the entries of the library that the package has loaded; torch's current stream of a device, as a number; what turns a
// code into an exception; the package's own exception
decltype(&sq_rope_kv_write_paged) entry_write;
decltype(&sq_kv_read_paged) entry_read;
decltype(&sq_paged_attention_workspace_bytes) entry_attention_bytes;
decltype(&sq_paged_attention) entry_attention;
decltype(&sq_verify_drafts_workspace_bytes) entry_verify_bytes;
decltype(&sq_verify_drafts) entry_verify;
PyObject *raw_stream, *check_code, *native_error;

struct Refused { PyObject* type; std::string what; };
[[noreturn]] void refuse(PyObject* type, const std::string& what) { throw Refused{type, what}; }

std::string text(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}
std::string text(ScalarType t) {
    switch (t) {
        case ScalarType::Half: return "torch.float16";
        case ScalarType::BFloat16: return "torch.bfloat16";
        case ScalarType::Float: return "torch.float32";
        case ScalarType::Float8_e4m3fn: return "torch.float8_e4m3fn";
        case ScalarType::Byte: return "torch.uint8";
        case ScalarType::Int: return "torch.int32";
        case ScalarType::Long: return "torch.int64";
        default: return c10::toString(t);
    }
}

const Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + ": expected a tensor, got " + Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
int whole(PyObject* o, const char* name) {
    const int64_t v = PyLong_Check(o) ? PyLong_AsLongLong(o) : [&] {
        PyObject* i = PyNumber_Index(o);
        if (!i) throw python_error();
        const int64_t w = PyLong_AsLongLong(i);
        Py_DECREF(i);
        return w;
    }();
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v < std::numeric_limits<int>::min() || v > std::numeric_limits<int>::max()) refuse(PyExc_ValueError, std::string(name) + ": " + std::to_string(v) + " is too large");
    return (int)v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
int narrow(int64_t v, const char* name) {
    if (v > std::numeric_limits<int>::max()) refuse(PyExc_ValueError, std::string(name) + ": " + std::to_string(v) + " are too many");
    return (int)v;
}

// the device of the call; every other tensor has to live there
struct Where {
    const at::Device device;
    explicit Where(const Tensor& first) : device(first.device()) {
        if (!device.is_cuda())
            refuse(native_error, "the tensors live on " + device.str() + ": the paged path only runs on a HIP device (no CPU fallback)");
    }
    void same(const Tensor& t) const {
        if (t.device() != device) refuse(PyExc_ValueError, "the call's tensors live on different devices: " + t.device().str() + " beside " + device.str());
    }
    void* stream() const {
        PyObject* const index = PyLong_FromLong(device.index());
        PyObject* const s = index ? PyObject_CallOneArg(raw_stream, index) : nullptr;
        Py_XDECREF(index);
        if (!s) throw python_error();
        void* const p = PyLong_AsVoidPtr(s);
        Py_DECREF(s);
        if (PyErr_Occurred()) throw python_error();
        return p;
    }
};

const Tensor& here(PyObject* o, const char* name, const Where& w) {
    const Tensor& t = tensor(o, name);
    w.same(t);
    return t;
}
// n contiguous entries
template <typename T> T* entries(PyObject* o, ScalarType type, int64_t n, const char* name, const Where& w) {
    const Tensor& t = here(o, name, w);
    if (t.scalar_type() != type) refuse(PyExc_TypeError, std::string(name) + ": expected " + text(type) + ", got " + text(t.scalar_type()));
    if (t.dim() != 1 || t.size(0) < n || !t.is_contiguous())
        refuse(PyExc_ValueError, std::string(name) + ": expected " + std::to_string(n) + " contiguous entries, got " + text(t));
    return (T*)t.data_ptr();
}

int half_code(const Tensor& t, const char* name) {
    if (t.scalar_type() == ScalarType::Half) return SQ_DTYPE_F16;
    if (t.scalar_type() == ScalarType::BFloat16) return SQ_DTYPE_BF16;
    refuse(PyExc_TypeError, std::string(name) + ": expected torch.float16 or torch.bfloat16, got " + text(t.scalar_type()));
}

// one layer's pages and the batch's table
struct Pool {
    void *k, *v, *ks = nullptr, *vs = nullptr;
    const int32_t* table;
    int n_pages, h_kv, page, d, n_seqs, width;
    Pool(PyObject* k_pages, PyObject* v_pages, PyObject* k_scales, PyObject* v_scales, PyObject* page_table, ScalarType type, const Where& w) {
        const Tensor &kp = here(k_pages, "k_pages", w), &vp = here(v_pages, "v_pages", w);
        if (kp.dim() != 4 || vp.sizes() != kp.sizes())
            refuse(PyExc_ValueError, "k_pages / v_pages: expected [n_pages, H_kv, page_size, D] twice, got " + text(kp) + ", " + text(vp));
        const bool quantised = k_scales != Py_None;
        if (quantised != (v_scales != Py_None)) refuse(PyExc_ValueError, "k_scales / v_scales: both or none");
        const ScalarType want = quantised ? ScalarType::Float8_e4m3fn : type;
        if (kp.scalar_type() != want || vp.scalar_type() != want)
            refuse(PyExc_TypeError, "k_pages / v_pages: expected " + text(want) + ", got " + text(kp.scalar_type()) + ", " + text(vp.scalar_type()));
        if (!kp.is_contiguous() || !vp.is_contiguous()) refuse(PyExc_ValueError, "k_pages / v_pages: must be contiguous");
        n_pages = narrow(kp.size(0), "pages"); h_kv = narrow(kp.size(1), "heads"); page = narrow(kp.size(2), "rows a page"); d = narrow(kp.size(3), "columns");
        k = kp.data_ptr(); v = vp.data_ptr();
        if (quantised) {
            ks = scales(k_scales, "k_scales", kp, w);
            vs = scales(v_scales, "v_scales", kp, w);
        }
        const Tensor& t = here(page_table, "page_table", w);
        if (t.scalar_type() != ScalarType::Int) refuse(PyExc_TypeError, "page_table: expected torch.int32, got " + text(t.scalar_type()));
        if (t.dim() != 2 || !t.is_contiguous()) refuse(PyExc_ValueError, "page_table: expected [sequences, pages] contiguous, got " + text(t));
        n_seqs = narrow(t.size(0), "sequences"); width = narrow(t.size(1), "pages a sequence");
        table = (const int32_t*)t.data_ptr();
    }
    static void* scales(PyObject* o, const char* name, const Tensor& pages, const Where& w) {
        const Tensor& t = here(o, name, w);
        if (t.scalar_type() != ScalarType::Byte) refuse(PyExc_TypeError, std::string(name) + ": expected torch.uint8, got " + text(t.scalar_type()));
        if (t.sizes() != pages.sizes().slice(0, 3) || !t.is_contiguous())
            refuse(PyExc_ValueError, std::string(name) + ": expected the pages' first three dimensions, contiguous, got " + text(t) + " for " + text(pages));
        return t.data_ptr();
    }
};

// One buffer a call, from the stream-ordered allocator: two streams or two captured graphs never share it, and what is allocated
// next gets its bytes behind this call's work.
Tensor workspace(size_t bytes, const Where& w) {
    return bytes ? at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(w.device)) : Tensor();
}
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

PyObject* finish(int code, const char* what) {
    if (code == SQ_OK) Py_RETURN_NONE;
    return PyObject_CallFunction(check_code, "is", code, what);
}

template <PyObject* (*CALL)(PyObject* const*), int ARGS> PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != ARGS) { PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", ARGS, n); return nullptr; }
    try {
        return CALL(args);
    } catch (const Refused& r) {
        PyErr_SetString(r.type, r.what.c_str());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// (qkv, q_out, k_pages, v_pages, cos, sin, position_ids, page_table, seq_lens, cu_rows, n_heads, h_kv, d, k_scales, v_scales)
PyObject* write(PyObject* const* a) {
    const Tensor& qkv = tensor(a[0], "qkv");
    const Where w(qkv);
    const int code = half_code(qkv, "qkv"), n_heads = whole(a[10], "n_heads"), h_kv = whole(a[11], "h_kv"), d = whole(a[12], "d");
    const Tensor &q_out = here(a[1], "q_out", w), &cos = here(a[4], "cos", w), &sin = here(a[5], "sin", w);
    const ScalarType type = qkv.scalar_type();
    if (q_out.scalar_type() != type || cos.scalar_type() != type || sin.scalar_type() != type)
        refuse(PyExc_TypeError, "q_out / cos / sin: expected " + text(type) + " three times, got " + text(q_out.scalar_type()) + ", " +
                                    text(cos.scalar_type()) + ", " + text(sin.scalar_type()));
    const Pool P(a[2], a[3], a[13], a[14], a[7], type, w);
    const int64_t cols = ((int64_t)n_heads + 2 * (int64_t)h_kv) * d;
    if (qkv.dim() != 2 || qkv.stride(1) != 1 || qkv.size(1) != cols || P.h_kv != h_kv || P.d != d)
        refuse(PyExc_ValueError, "qkv: expected [n_rows, " + std::to_string(cols) + "] with unit inner stride over pages of " + std::to_string(h_kv) +
                                     " heads of " + std::to_string(d) + ", got " + text(qkv) + " over " + std::to_string(P.h_kv) + " heads of " + std::to_string(P.d));
    const int n_rows = narrow(qkv.size(0), "rows");
    if (q_out.dim() != 3 || q_out.size(0) != n_heads || q_out.size(1) != n_rows || q_out.size(2) != d || !q_out.is_contiguous())
        refuse(PyExc_ValueError, "q_out: expected [" + std::to_string(n_heads) + ", " + std::to_string(n_rows) + ", " + std::to_string(d) + "] contiguous, got " + text(q_out));
    if (cos.dim() != 2 || cos.size(1) != d || sin.sizes() != cos.sizes() || !cos.is_contiguous() || !sin.is_contiguous())
        refuse(PyExc_ValueError, "cos / sin: expected [positions, " + std::to_string(d) + "] contiguous twice, got " + text(cos) + ", " + text(sin));
    const auto* pos = entries<int64_t>(a[6], ScalarType::Long, n_rows, "position_ids", w);
    const auto* lens = entries<int32_t>(a[8], ScalarType::Int, P.n_seqs, "seq_lens", w);
    const auto* cu = entries<int32_t>(a[9], ScalarType::Int, (int64_t)P.n_seqs + 1, "cu_rows", w);
    const c10::OptionalDeviceGuard current(w.device);
    return finish(entry_write(qkv.data_ptr(), n_rows > 1 ? qkv.stride(0) : cols, q_out.data_ptr(), P.k, P.v, P.ks, P.vs, cos.data_ptr(), sin.data_ptr(),
                              narrow(cos.size(0), "positions"), pos, P.table, P.width, P.n_pages, P.page, lens, cu, P.n_seqs, n_rows, n_heads, h_kv, d,
                              code, w.stream()),
                  "sq_rope_kv_write_paged");
}

// (k_pages, v_pages, k_out, v_out, page_table, starts, counts, max_count, k_scales, v_scales)
PyObject* read(PyObject* const* a) {
    const Tensor& k_out = tensor(a[2], "k_out");
    const Where w(k_out);
    const Tensor& v_out = here(a[3], "v_out", w);
    const int code = half_code(k_out, "k_out");
    if (v_out.scalar_type() != k_out.scalar_type())
        refuse(PyExc_TypeError, "v_out: expected " + text(k_out.scalar_type()) + ", got " + text(v_out.scalar_type()));
    const Pool P(a[0], a[1], a[8], a[9], a[4], k_out.scalar_type(), w);
    if (k_out.dim() != 4 || k_out.size(0) != P.n_seqs || k_out.size(1) != P.h_kv || k_out.size(3) != P.d || v_out.sizes() != k_out.sizes())
        refuse(PyExc_ValueError, "k_out / v_out: expected [" + std::to_string(P.n_seqs) + ", " + std::to_string(P.h_kv) + ", M, " + std::to_string(P.d) +
                                     "] twice, got " + text(k_out) + ", " + text(v_out));
    const int m = narrow(k_out.size(2), "rows");
    const int64_t plane = (int64_t)m * P.d;
    const auto s = k_out.strides();
    if (v_out.strides() != s || s[3] != 1 || (m > 1 && s[2] != P.d) || (P.h_kv > 1 && s[1] < plane) || (P.n_seqs > 1 && s[0] < plane))
        refuse(PyExc_ValueError, "k_out / v_out: expected contiguous rows and the same strides, got " + text(k_out) + " with other ones");
    const auto* starts = entries<int32_t>(a[5], ScalarType::Int, P.n_seqs, "starts", w);
    const auto* counts = entries<int32_t>(a[6], ScalarType::Int, P.n_seqs, "counts", w);
    const int most = a[7] == Py_None ? m : whole(a[7], "max_count");
    if (most < 0 || most > m) refuse(PyExc_ValueError, "max_count: " + std::to_string(most) + " is not between 0 and " + std::to_string(m));
    const c10::OptionalDeviceGuard current(w.device);
    return finish(entry_read(P.k, P.v, P.ks, P.vs, k_out.data_ptr(), v_out.data_ptr(), P.n_seqs > 1 ? s[0] : P.h_kv * plane, P.h_kv > 1 ? s[1] : plane, m,
                             P.table, P.width, P.n_pages, P.page, starts, counts, P.n_seqs, most, P.h_kv, P.d, code, w.stream()),
                  "sq_kv_read_paged");
}

// (q, k_pages, v_pages, out, page_table, seq_lens, cu_rows, scale, max_rows, max_len, k_scales, v_scales)
PyObject* attention(PyObject* const* a) {
    const Tensor& q = tensor(a[0], "q");
    const Where w(q);
    const Tensor& out = here(a[3], "out", w);
    const int code = half_code(q, "q");
    if (out.scalar_type() != q.scalar_type()) refuse(PyExc_TypeError, "out: expected " + text(q.scalar_type()) + ", got " + text(out.scalar_type()));
    const Pool P(a[1], a[2], a[10], a[11], a[4], q.scalar_type(), w);
    if (q.dim() != 3 || q.size(2) != P.d || !P.h_kv || q.size(0) % P.h_kv || q.stride(2) != 1)
        refuse(PyExc_ValueError, "q: expected [H, n_rows, " + std::to_string(P.d) + "] with unit inner stride and a multiple of " + std::to_string(P.h_kv) +
                                     " heads, got " + text(q));
    const int n_heads = narrow(q.size(0), "heads"), n_rows = narrow(q.size(1), "rows");
    const int64_t cols = (int64_t)n_heads * P.d;
    if (out.dim() != 2 || out.size(0) != n_rows || out.size(1) != cols || out.stride(1) != 1 || (n_rows > 1 && out.stride(0) < cols))
        refuse(PyExc_ValueError, "out: expected [" + std::to_string(n_rows) + ", " + std::to_string(cols) + "] with unit inner stride, got " + text(out));
    const auto* lens = entries<int32_t>(a[5], ScalarType::Int, P.n_seqs, "seq_lens", w);
    const auto* cu = entries<int32_t>(a[6], ScalarType::Int, (int64_t)P.n_seqs + 1, "cu_rows", w);
    int64_t max_rows = a[8] == Py_None ? n_rows : whole(a[8], "max_rows"), max_len = (int64_t)P.width * P.page;
    if (a[9] != Py_None) max_len = std::min<int64_t>(whole(a[9], "max_len"), max_len);
    if (max_rows < 0 || max_len < 0)
        refuse(PyExc_ValueError, "max_rows " + std::to_string(max_rows) + " / max_len " + std::to_string(max_len) + ": expected bounds >= 0");
    max_rows = std::min<int64_t>(max_rows, n_rows);
    const int keys = narrow(max_len, "keys");
    const double scale = number(a[7]);
    if (!(scale > 0.0 && scale < std::numeric_limits<double>::infinity())) refuse(PyExc_ValueError, "scale: expected a positive number, got " + std::to_string(scale));
    const c10::OptionalDeviceGuard current(w.device);
    const size_t need = entry_attention_bytes(P.n_seqs, n_rows, (int)max_rows, keys, n_heads, P.h_kv, P.d);
    const Tensor ws = workspace(need, w);
    return finish(entry_attention(q.data_ptr(), n_heads > 1 ? q.stride(0) : 0, n_rows > 1 ? q.stride(1) : 0, P.k, P.v, P.ks, P.vs, out.data_ptr(),
                                  n_rows > 1 ? out.stride(0) : cols, P.table, P.width, P.n_pages, P.page, lens, cu, P.n_seqs, n_rows, (int)max_rows, keys,
                                  n_heads, P.h_kv, P.d, (float)scale, code, pointer(ws), need, w.stream()),
                  "sq_paged_attention");
}

// (target_logits, draft_logits, draft_tokens, cu_drafts, u_accept, u_next, temperature, n_accepted, next_tokens)
PyObject* verify(PyObject* const* a) {
    const Tensor& target = tensor(a[0], "target_logits");
    const Where w(target);
    const Tensor &draft = here(a[1], "draft_logits", w), &tokens = here(a[2], "draft_tokens", w), &accepted = here(a[7], "n_accepted", w);
    const ScalarType type = target.scalar_type();
    const int code = type == ScalarType::Half ? SQ_DTYPE_F16 : type == ScalarType::BFloat16 ? SQ_DTYPE_BF16 : SQ_DTYPE_F32;
    if ((code == SQ_DTYPE_F32 && type != ScalarType::Float) || draft.scalar_type() != type)
        refuse(PyExc_TypeError, "target_logits / draft_logits: expected fp16, bf16 or fp32 twice, got " + text(type) + ", " + text(draft.scalar_type()));
    if (tokens.dim() != 1 || accepted.dim() != 1)
        refuse(PyExc_ValueError, "draft_tokens / n_accepted: expected one dimension, got " + text(tokens) + ", " + text(accepted));
    const int n_seqs = narrow(accepted.size(0), "sequences"), n_drafts = narrow(tokens.size(0), "drafted tokens");
    if (target.dim() != 2 || draft.dim() != 2 || target.size(1) != draft.size(1))
        refuse(PyExc_ValueError, "target_logits / draft_logits: expected two dimensions and one vocabulary, got " + text(target) + ", " + text(draft));
    const int64_t vocab = target.size(1);
    const auto rows = [&](const Tensor& t, int64_t n, const char* name) {
        if (t.size(0) < n || (n && t.stride(1) != 1) || (n > 1 && t.stride(0) < vocab))
            refuse(PyExc_ValueError, std::string(name) + ": expected " + std::to_string(n) + " rows with unit inner stride, got " + text(t));
        return std::max(t.stride(0), vocab);
    };
    const int64_t ld_t = rows(target, (int64_t)n_drafts + n_seqs, "target_logits"), ld_d = rows(draft, n_drafts, "draft_logits");
    const auto* tok = entries<int64_t>(a[2], ScalarType::Long, n_drafts, "draft_tokens", w);
    const auto* cu = entries<int32_t>(a[3], ScalarType::Int, (int64_t)n_seqs + 1, "cu_drafts", w);
    const auto* ua = entries<float>(a[4], ScalarType::Float, n_drafts, "u_accept", w);
    const auto* un = entries<float>(a[5], ScalarType::Float, n_seqs, "u_next", w);
    auto* acc = entries<int32_t>(a[7], ScalarType::Int, n_seqs, "n_accepted", w);
    auto* next = entries<int64_t>(a[8], ScalarType::Long, n_seqs, "next_tokens", w);
    const float* temps = nullptr;
    double temp = 0.0;
    if (THPVariable_Check(a[6])) {
        temps = entries<float>(a[6], ScalarType::Float, n_seqs, "temperature", w);
    } else {
        temp = number(a[6]);
        if (!(temp >= 0.0 && temp < std::numeric_limits<double>::infinity()))
            refuse(PyExc_ValueError, "temperature: expected a number >= 0, got " + std::to_string(temp));
    }
    const c10::OptionalDeviceGuard current(w.device);
    const int v = narrow(vocab, "tokens of the vocabulary");
    const size_t need = entry_verify_bytes(n_seqs, n_drafts, v);
    const Tensor ws = workspace(need, w);
    return finish(entry_verify(target.data_ptr(), ld_t, draft.data_ptr(), ld_d, tok, cu, n_seqs, n_drafts, v, ua, un, temps, (float)temp, acc, next, code,
                               pointer(ws), need, w.stream()),
                  "sq_verify_drafts");
}

// (addresses of the six entries, raw_stream, check, SequoiaNativeError)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long at[6];
    PyObject *s, *c, *e;
    if (!PyArg_ParseTuple(args, "KKKKKKOOO", &at[0], &at[1], &at[2], &at[3], &at[4], &at[5], &s, &c, &e)) return nullptr;
    entry_write = (decltype(entry_write))at[0];
    entry_read = (decltype(entry_read))at[1];
    entry_attention_bytes = (decltype(entry_attention_bytes))at[2];
    entry_attention = (decltype(entry_attention))at[3];
    entry_verify_bytes = (decltype(entry_verify_bytes))at[4];
    entry_verify = (decltype(entry_verify))at[5];
    for (PyObject* o : {s, c, e}) Py_INCREF(o);              // kept as long as the process
    raw_stream = s; check_code = c; native_error = e;
    Py_RETURN_NONE;
}

#define SQ_METHOD(NAME, ARGS) {#NAME, (PyCFunction)(void (*)(void))(guarded<NAME, ARGS>), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {SQ_METHOD(write, 15), SQ_METHOD(read, 10), SQ_METHOD(attention, 12), SQ_METHOD(verify, 9),
                         {"bind", bind, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged() { return PyModule_Create(&module); }
