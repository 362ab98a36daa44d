// The text decoder's calls on torch tensors without the interpreter in between: ocrhip._tensors reads
// a tensor's type, shape, strides and address itself and calls the library. A step of single tokens
// takes a handful of calls of a few microseconds of GPU work each, which Python's own checks of their
// arrays (0.9 us an array) outlast.
//
// It takes only what is right in every respect: arguments that are not answer kOther, and the
// caller's checks in Python say what is wrong with them (or deal with arrays that are no tensors).
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "../../../include/ocrhip.h"

namespace {

constexpr long kOther = -2;
constexpr int kI32 = 5;  // beside OCR_F32 ... OCR_E4M3
constexpr unsigned F32 = 1 << OCR_F32, HALVES = 1 << OCR_F16 | 1 << OCR_BF16, I32 = 1 << kI32;

// The library's functions, by address: it is loaded by its path, under no name that a linker knows.
decltype(&ocr_kv_append_device) g_append;
decltype(&ocr_kv_read_device) g_read;
decltype(&ocr_attention_device) g_attention;
decltype(&ocr_decode_attention_device) g_decode;
decltype(&ocr_beam_select_device) g_beam;
decltype(&ocr_kv_fork_device) g_fork;

struct Call {
    bool ok = true;
    int device;

    const at::Tensor *tensor(PyObject *o, unsigned types, int *code = nullptr) {
        if (!THPVariable_Check(o)) return no();
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.get_device() != device || t.layout() != at::kStrided) return no();
        int c;
        switch (t.scalar_type()) {
            case at::kFloat: c = OCR_F32; break;
            case at::kHalf: c = OCR_F16; break;
            case at::kBFloat16: c = OCR_BF16; break;
            case at::kInt: c = kI32; break;
            default: return no();
        }
        if (!(types >> c & 1)) return no();
        if (code) *code = c;
        return &t;
    }
    // An array of exactly these sizes, its values one after another; None is NULL where it may be.
    void *flat(PyObject *o, unsigned types, std::initializer_list<int64_t> sizes, bool optional = false, int *code = nullptr) {
        if (optional && o == Py_None) return nullptr;
        const at::Tensor *t = tensor(o, types, code);
        if (!t || t->sizes() != at::IntArrayRef(sizes.begin(), sizes.size()) || !t->is_contiguous()) return no();
        return t->data_ptr();
    }
    // [tokens][heads][dim] whose tokens may lie apart; sizes under 0 take what is there.
    void *tokens(PyObject *o, unsigned types, int64_t *n, int64_t *heads, int64_t *dim, int64_t *stride, int *code) {
        const at::Tensor *t = tensor(o, types, code);
        if (!t || t->dim() != 3) return no();
        int64_t *want[3] = {n, heads, dim};
        for (int k = 0; k < 3; k++) {
            if (*want[k] >= 0 && *want[k] != t->size(k)) return no();
            *want[k] = t->size(k);
            if (t->size(k) < 1) return no();
        }
        if ((*dim > 1 && t->stride(2) != 1) || (*heads > 1 && t->stride(1) != *dim)) return no();
        *stride = *n > 1 ? t->stride(0) : *heads * *dim;
        return t->data_ptr();
    }
    // [rows][values] whose rows may lie apart.
    void *rows(PyObject *o, unsigned types, int64_t *n, int64_t *width, int64_t *stride, int *code) {
        const at::Tensor *t = tensor(o, types, code);
        if (!t || t->dim() != 2 || t->size(0) < 1 || t->size(1) < 1 || (t->size(1) > 1 && t->stride(1) != 1)) return no();
        if ((*n >= 0 && *n != t->size(0)) || (*width >= 0 && *width != t->size(1))) return no();
        *n = t->size(0), *width = t->size(1);
        *stride = *n > 1 ? t->stride(0) : *width;
        return t->data_ptr();
    }
    ocr_page_table table(PyObject *o) {
        const at::Tensor *t = tensor(o, I32);
        if (!t || t->dim() != 2 || !t->is_contiguous()) {
            no();
            return {};
        }
        fits(t->size(0)), fits(t->size(1));
        return {static_cast<const int32_t *>(t->data_ptr()), uint32_t(t->size(0)), uint32_t(t->size(1))};
    }
    std::nullptr_t no() {
        ok = false;
        return nullptr;
    }
    void fits(int64_t v) { ok = ok && v >= 0 && v <= INT32_MAX; }
    int64_t whole(PyObject *o) {
        const int64_t v = PyLong_CheckExact(o) ? PyLong_AsLongLong(o) : -1;
        if (v < 0) PyErr_Clear(), no();
        return v;
    }
    double real(PyObject *o) {
        if (!PyFloat_Check(o) && !PyLong_CheckExact(o)) no();
        const double v = ok ? PyFloat_AsDouble(o) : 0;
        if (PyErr_Occurred()) PyErr_Clear(), no();
        return v;
    }
    template <class T> T *address(PyObject *o) {
        void *p = PyLong_CheckExact(o) ? PyLong_AsVoidPtr(o) : nullptr;
        if (!p) PyErr_Clear(), no();
        return static_cast<T *>(p);
    }
};

template <class F> PyObject *done(const Call &c, F &&f) {
    long rc = kOther;
    if (c.ok) {
        Py_BEGIN_ALLOW_THREADS
        rc = f();
        Py_END_ALLOW_THREADS
    }
    return PyLong_FromLong(rc);
}
bool count_is(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return n == want;
}
#define OCR_CALL(name, n) PyObject *name(PyObject *, PyObject *const *v, Py_ssize_t count) try { \
    if (!count_is(count, n)) return nullptr; \
    Call c; \
    ocr_ctx *const ctx = c.address<ocr_ctx>(v[0]); \
    c.device = int(c.whole(v[1]));
// Nothing above throws on tensors that it takes; what does is not dealt with here.
#define OCR_END } catch (...) { return PyLong_FromLong(kOther); }

// handle, device, cache, table, seq, pos, qkv, q, k, q_norm, k_norm, eps, rot, theta, adjacent
OCR_CALL(append, 15)
    const auto *cache = c.address<const ocr_kv_cache>(v[2]);
    if (!c.ok) return PyLong_FromLong(kOther);
    const ocr_page_table table = c.table(v[3]);
    ocr_kv_append_args a{};
    int64_t n = -1, q_heads = -1, dim = cache->dim, q_stride = 0;
    a.q = c.tokens(v[7], HALVES, &n, &q_heads, &dim, &q_stride, &a.out_type);
    if (!c.ok || q_stride != q_heads * dim) return PyLong_FromLong(kOther);
    int64_t rows = n, width = (q_heads + 2 * int64_t(cache->heads)) * dim;
    a.qkv = c.rows(v[6], F32 | HALVES, &rows, &width, &a.stride, &a.type);
    a.seq = static_cast<const int32_t *>(c.flat(v[4], I32, {n}));
    a.pos = static_cast<const int32_t *>(c.flat(v[5], I32, {n}));
    a.k = c.flat(v[8], 1u << a.out_type, {n, int64_t(cache->heads), dim}, true);
    a.q_norm = static_cast<const float *>(c.flat(v[9], F32, {dim}, true));
    a.k_norm = static_cast<const float *>(c.flat(v[10], F32, {dim}, true));
    a.eps = float(c.real(v[11])), a.rot = uint32_t(c.whole(v[12])), a.theta = c.real(v[13]), a.adjacent = v[14] == Py_True;
    a.n = uint32_t(n), a.q_heads = uint32_t(q_heads);
    c.fits(n), c.fits(q_heads);
    if (!(a.theta > 0)) c.no();
    return done(c, [&] { return g_append(ctx, cache, &table, &a); });
OCR_END

// handle, device, cache, table, lens, k, v
OCR_CALL(read, 7)
    const auto *cache = c.address<const ocr_kv_cache>(v[2]);
    const at::Tensor *k = c.tensor(v[5], HALVES);
    if (!c.ok || k->dim() != 4) return PyLong_FromLong(kOther);
    const ocr_page_table table = c.table(v[3]);
    const int64_t most = k->size(1);
    const std::initializer_list<int64_t> shape = {int64_t(table.rows), most, int64_t(cache->heads), int64_t(cache->dim)};
    int type = 0;
    void *kp = c.flat(v[5], HALVES, shape, false, &type), *vp = c.flat(v[6], 1u << type, shape);
    const auto *lens = static_cast<const int32_t *>(c.flat(v[4], I32, {int64_t(table.rows)}));
    c.fits(most);
    return done(c, [&] { return g_read(ctx, cache, &table, lens, uint32_t(most), type, kp, vp); });
OCR_END

// handle, device, cache, table, lens, q, out, scale, cap, slopes
OCR_CALL(attend, 10)
    const auto *cache = c.address<const ocr_kv_cache>(v[2]);
    if (!c.ok) return PyLong_FromLong(kOther);
    const ocr_page_table table = c.table(v[3]);
    ocr_decode_args a{};
    int64_t n = table.rows, q_heads = -1, dim = cache->dim;
    int code = 0;
    a.q = c.tokens(v[5], HALVES, &n, &q_heads, &dim, &a.q_stride, &a.type);
    a.out = c.tokens(v[6], 1u << a.type, &n, &q_heads, &dim, &a.out_stride, &code);
    a.lens = static_cast<const int32_t *>(c.flat(v[4], I32, {n}));
    a.q_heads = uint32_t(q_heads), a.scale = float(c.real(v[7])), a.cap = float(c.real(v[8]));
    a.slopes = static_cast<const float *>(c.flat(v[9], F32, {q_heads}, true));
    c.fits(q_heads);
    return done(c, [&] { return g_decode(ctx, cache, &table, &a); });
OCR_END

// handle, device, cache, table, lens, parents, spare, table_out, lens_out, used
OCR_CALL(fork, 10)
    const auto *cache = c.address<const ocr_kv_cache>(v[2]);
    const ocr_page_table table = c.table(v[3]);
    const at::Tensor *parents = c.tensor(v[5], I32);
    if (!c.ok || parents->dim() != 2 || !parents->is_contiguous() || parents->numel() != int64_t(table.rows)) return PyLong_FromLong(kOther);
    auto ints = [&](PyObject *o, std::initializer_list<int64_t> sizes) { return static_cast<int32_t *>(c.flat(o, I32, sizes)); };
    const int64_t rows = table.rows;
    const int32_t *lens = ints(v[4], {rows}), *spare = ints(v[6], {rows}), *from = static_cast<const int32_t *>(parents->data_ptr());
    int32_t *table_out = ints(v[7], {rows, int64_t(table.width)}), *lens_out = ints(v[8], {rows}), *used = ints(v[9], {rows});
    const uint32_t beams = uint32_t(parents->size(1));
    return done(c, [&] { return g_fork(ctx, cache, &table, lens, from, beams, spare, table_out, lens_out, used); });
OCR_END

// handle, device, q, k, v, out, docs, prefix, scale, cap, slopes
OCR_CALL(attention, 11)
    ocr_attention_args a{};
    int64_t n = -1, q_heads = -1, kv_heads = -1, dim = -1;
    int code = 0;
    a.q = c.tokens(v[2], HALVES, &n, &q_heads, &dim, &a.q_stride, &a.type);
    a.k = c.tokens(v[3], 1u << a.type, &n, &kv_heads, &dim, &a.k_stride, &code);
    a.v = c.tokens(v[4], 1u << a.type, &n, &kv_heads, &dim, &a.v_stride, &code);
    a.out = c.tokens(v[5], 1u << a.type, &n, &q_heads, &dim, &a.out_stride, &code);
    int64_t ndocs = 1;
    if (v[6] != Py_None) {
        const at::Tensor *docs = c.tensor(v[6], I32);
        if (!c.ok || docs->dim() != 1 || docs->size(0) < 1 || !docs->is_contiguous()) return PyLong_FromLong(kOther);
        ndocs = docs->size(0) - 1;
        a.docs = static_cast<const int32_t *>(docs->data_ptr());
    }
    a.ndocs = uint32_t(ndocs);
    a.prefix = static_cast<const int32_t *>(c.flat(v[7], I32, {ndocs}, true));
    a.slopes = static_cast<const float *>(c.flat(v[10], F32, {q_heads}, true));
    a.n = uint32_t(n), a.q_heads = uint32_t(q_heads), a.kv_heads = uint32_t(kv_heads), a.dim = uint32_t(dim);
    a.scale = float(c.real(v[8])), a.cap = float(c.real(v[9]));
    c.fits(n), c.fits(q_heads), c.fits(kv_heads), c.fits(dim), c.fits(ndocs);
    return done(c, [&] { return g_attention(ctx, &a); });
OCR_END

// handle, device, logits, scores, finished, eos, out_scores, parents, tokens, out_finished
OCR_CALL(beam_select, 10)
    const at::Tensor *scores = c.tensor(v[3], F32);
    if (!c.ok || scores->dim() != 2) return PyLong_FromLong(kOther);
    const int64_t groups = scores->size(0), beams = scores->size(1);
    ocr_beam_args a{};
    int64_t rows = groups * beams, vocab = -1;
    a.logits = c.rows(v[2], F32 | HALVES, &rows, &vocab, &a.stride, &a.type);
    auto ints = [&](PyObject *o, bool optional) { return static_cast<int32_t *>(c.flat(o, I32, {groups, beams}, optional)); };
    a.scores = static_cast<const float *>(c.flat(v[3], F32, {groups, beams}));
    a.finished = ints(v[4], true);
    a.eos = v[5] == Py_None ? -1 : int32_t(c.whole(v[5]));
    a.out_scores = static_cast<float *>(c.flat(v[6], F32, {groups, beams}));
    a.parents = ints(v[7], false), a.tokens = ints(v[8], false), a.out_finished = ints(v[9], true);
    a.groups = uint32_t(groups), a.beams = uint32_t(beams), a.vocab = uint32_t(vocab);
    c.fits(groups), c.fits(beams), c.fits(vocab);
    if (v[5] != Py_None) c.fits(c.whole(v[5]));
    return done(c, [&] { return g_beam(ctx, &a); });
OCR_END

// The six functions' addresses, in the order of the pointers above.
PyObject *bind(PyObject *, PyObject *const *v, Py_ssize_t count) {
    if (!count_is(count, 6)) return nullptr;
    void *p[6];
    for (int k = 0; k < 6; k++)
        if (!(p[k] = PyLong_AsVoidPtr(v[k]))) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no address");
            return nullptr;
        }
    g_append = reinterpret_cast<decltype(g_append)>(p[0]), g_read = reinterpret_cast<decltype(g_read)>(p[1]);
    g_attention = reinterpret_cast<decltype(g_attention)>(p[2]), g_decode = reinterpret_cast<decltype(g_decode)>(p[3]);
    g_beam = reinterpret_cast<decltype(g_beam)>(p[4]), g_fork = reinterpret_cast<decltype(g_fork)>(p[5]);
    Py_RETURN_NONE;
}

#define OCR_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {OCR_METHOD(bind), OCR_METHOD(append), OCR_METHOD(read), OCR_METHOD(attend), OCR_METHOD(fork),
                         OCR_METHOD(attention), OCR_METHOD(beam_select), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
