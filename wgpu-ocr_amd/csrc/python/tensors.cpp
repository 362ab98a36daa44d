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
decltype(&ocr_kv_append_axes_device) g_append_axes;
decltype(&ocr_rotate_device) g_rotate;
decltype(&ocr_attention_weights_device) g_attention_weights;
decltype(&ocr_decode_attention_weights_device) g_decode_weights;
decltype(&ocr_kv_evict_device) g_evict;
decltype(&ocr_latent_append_device) g_latent_append;
decltype(&ocr_latent_decode_device) g_latent_decode;
decltype(&ocr_latent_attention_device) g_latent_attention;

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
    // The same with heads that may lie apart too.
    void *heads(PyObject *o, unsigned types, int64_t *n, int64_t *count, int64_t *dim, int64_t *stride, int64_t *head, int *code) {
        const at::Tensor *t = tensor(o, types, code);
        if (!t || t->dim() != 3) return no();
        int64_t *want[3] = {n, count, dim};
        for (int k = 0; k < 3; k++) {
            if (*want[k] >= 0 && *want[k] != t->size(k)) return no();
            *want[k] = t->size(k);
            if (t->size(k) < 1) return no();
        }
        if (*dim > 1 && t->stride(2) != 1) return no();
        *head = *count > 1 ? t->stride(1) : *dim;
        *stride = *n > 1 ? t->stride(0) : (*count - 1) * *head + *dim;
        return t->data_ptr();
    }
    // Positions [n][axes] or [n], and the pairs of each axis (a tuple, or None for as many each).
    ocr_axes axes(PyObject *at, PyObject *pairs, int64_t n, int64_t rot, PyObject *in_turn, PyObject *own) {
        ocr_axes x{};
        const at::Tensor *t = tensor(at, I32);
        if (!t || t->dim() < 1 || t->dim() > 2 || t->size(0) != n || !t->is_contiguous()) return no(), x;
        const int64_t count = t->dim() == 2 ? t->size(1) : 1;
        if (count < 1 || count > 4) return no(), x;
        x.at = static_cast<const int32_t *>(t->data_ptr()), x.count = uint32_t(count);
        if (pairs == Py_None) {
            if (rot / 2 % count) return no(), x;
            for (int64_t k = 0; k < count; k++) x.pairs[k] = uint32_t(rot / 2 / count);
        } else {
            if (!PyTuple_CheckExact(pairs) || PyTuple_GET_SIZE(pairs) != count) return no(), x;
            for (int64_t k = 0; k < count; k++) {
                const int64_t v = whole(PyTuple_GET_ITEM(pairs, k));
                fits(v);
                x.pairs[k] = uint32_t(v);
            }
        }
        x.in_turn = in_turn == Py_True, x.own_ladder = own == Py_True;
        return x;
    }
    // [rows][heads][places], its places.
    void *places(PyObject *o, unsigned types, int64_t rows, int64_t count, int64_t *most) {
        const at::Tensor *t = tensor(o, types);
        if (!t || t->dim() != 3 || t->size(0) != rows || t->size(1) != count || !t->is_contiguous()) return no();
        *most = t->size(2);
        fits(*most);
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

// cache, table, seq, pos, qkv, q, k, q_norm, k_norm, eps, rot, theta, adjacent
bool append_args(Call &c, PyObject *const *v, const ocr_kv_cache *cache, ocr_kv_append_args &a) {
    int64_t n = -1, q_heads = -1, dim = cache->dim, q_stride = 0;
    a.q = c.tokens(v[5], HALVES, &n, &q_heads, &dim, &q_stride, &a.out_type);
    if (!c.ok || q_stride != q_heads * dim) return false;
    int64_t rows = n, width = (q_heads + 2 * int64_t(cache->heads)) * dim;
    a.qkv = c.rows(v[4], F32 | HALVES, &rows, &width, &a.stride, &a.type);
    a.seq = static_cast<const int32_t *>(c.flat(v[2], I32, {n}));
    a.pos = static_cast<const int32_t *>(c.flat(v[3], I32, {n}));
    a.k = c.flat(v[6], 1u << a.out_type, {n, int64_t(cache->heads), dim}, true);
    a.q_norm = static_cast<const float *>(c.flat(v[7], F32, {dim}, true));
    a.k_norm = static_cast<const float *>(c.flat(v[8], F32, {dim}, true));
    a.eps = float(c.real(v[9])), a.rot = uint32_t(c.whole(v[10])), a.theta = c.real(v[11]), a.adjacent = v[12] == Py_True;
    a.n = uint32_t(n), a.q_heads = uint32_t(q_heads);
    c.fits(n), c.fits(q_heads), c.fits(c.whole(v[10]));
    if (!(a.theta > 0)) c.no();
    return true;
}

// handle, device, and the above
OCR_CALL(append, 15)
    const auto *cache = c.address<const ocr_kv_cache>(v[2]);
    if (!c.ok) return PyLong_FromLong(kOther);
    const ocr_page_table table = c.table(v[3]);
    ocr_kv_append_args a{};
    if (!append_args(c, v + 2, cache, a)) return PyLong_FromLong(kOther);
    return done(c, [&] { return g_append(ctx, cache, &table, &a); });
OCR_END

// the above, at, axes, in_turn, own_ladder
OCR_CALL(append_axes, 19)
    const auto *cache = c.address<const ocr_kv_cache>(v[2]);
    if (!c.ok) return PyLong_FromLong(kOther);
    const ocr_page_table table = c.table(v[3]);
    ocr_kv_append_args a{};
    if (!append_args(c, v + 2, cache, a)) return PyLong_FromLong(kOther);
    const ocr_axes axes = c.axes(v[15], v[16], a.n, a.rot, v[17], v[18]);
    return done(c, [&] { return g_append_axes(ctx, cache, &table, &a, &axes); });
OCR_END

// handle, device, x, at, out, first, rot, theta, adjacent, axes, in_turn, own_ladder, back
OCR_CALL(rotate, 13)
    ocr_rotate_args a{};
    int64_t n = -1, heads = -1, dim = -1;
    int code = 0;
    a.x = c.heads(v[2], F32 | HALVES, &n, &heads, &dim, &a.x_stride, &a.x_head, &a.type);
    a.out = c.heads(v[4], 1u << a.type, &n, &heads, &dim, &a.out_stride, &a.out_head, &code);
    const int64_t first = c.whole(v[5]), rot = c.whole(v[6]);
    c.fits(n), c.fits(heads), c.fits(dim), c.fits(first), c.fits(rot);
    a.n = uint32_t(n), a.heads = uint32_t(heads), a.dim = uint32_t(dim), a.first = uint32_t(first), a.rot = uint32_t(rot);
    a.theta = c.real(v[7]), a.adjacent = v[8] == Py_True, a.back = v[12] == Py_True;
    if (!(a.theta > 0)) c.no();
    if (!c.ok) return PyLong_FromLong(kOther);
    const ocr_axes axes = c.axes(v[3], v[9], n, rot, v[10], v[11]);
    return done(c, [&] { return g_rotate(ctx, &a, &axes); });
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

// handle, device, cache, table, lens, q, out, scale, cap, slopes, weights
OCR_CALL(attend, 11)
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
    int64_t most = 0;
    float *weights = v[10] == Py_None ? nullptr : static_cast<float *>(c.places(v[10], F32, n, cache->heads, &most));
    return done(c, [&] { return weights ? g_decode_weights(ctx, cache, &table, &a, weights, uint32_t(most)) : g_decode(ctx, cache, &table, &a); });
OCR_END

// handle, device, cache, table, lens, newest, weights, held, keep, lens_out, first, recent, weights_out, held_out
OCR_CALL(evict, 14)
    const auto *cache = c.address<const ocr_kv_cache>(v[2]);
    if (!c.ok) return PyLong_FromLong(kOther);
    const ocr_page_table table = c.table(v[3]);
    const int64_t rows = table.rows, heads = cache->heads;
    int64_t most[4] = {};
    ocr_evict_args a{};
    auto ints = [&](PyObject *o) { return static_cast<int32_t *>(c.flat(o, I32, {rows})); };
    a.lens = ints(v[4]), a.newest = ints(v[5]), a.lens_out = ints(v[9]);
    a.weights = static_cast<const float *>(c.places(v[6], F32, rows, heads, &most[0]));
    a.held = static_cast<const int32_t *>(c.places(v[7], I32, rows, heads, &most[1]));
    a.weights_out = static_cast<float *>(c.places(v[12], F32, rows, heads, &most[2]));
    a.held_out = static_cast<int32_t *>(c.places(v[13], I32, rows, heads, &most[3]));
    const int64_t keep = c.whole(v[8]), first = c.whole(v[10]), recent = c.whole(v[11]);
    c.fits(keep), c.fits(first), c.fits(recent);
    if (most[1] != most[0] || most[2] != most[0] || most[3] != most[0]) c.no();
    a.most = uint32_t(most[0]), a.keep = uint32_t(keep), a.first = uint32_t(first), a.recent = uint32_t(recent);
    return done(c, [&] { return g_evict(ctx, cache, &table, &a); });
OCR_END

// handle, device, cache, table, seq, pos, x, out, norm, eps, theta, adjacent, at, axes, in_turn, own_ladder
OCR_CALL(latent_append, 16)
    const auto *cache = c.address<const ocr_latent_cache>(v[2]);
    if (!c.ok) return PyLong_FromLong(kOther);
    const ocr_page_table table = c.table(v[3]);
    ocr_latent_append_args a{};
    int64_t n = -1, width = int64_t(cache->rank) + cache->rot;
    a.x = c.rows(v[6], F32 | HALVES, &n, &width, &a.stride, &a.type);
    a.seq = static_cast<const int32_t *>(c.flat(v[4], I32, {n}));
    a.pos = static_cast<const int32_t *>(c.flat(v[5], I32, {n}));
    a.out = c.flat(v[7], 1u << cache->type, {n, width}, true);
    a.norm = static_cast<const float *>(c.flat(v[8], F32, {int64_t(cache->rank)}, true));
    a.eps = float(c.real(v[9])), a.theta = c.real(v[10]), a.adjacent = v[11] == Py_True, a.n = uint32_t(n);
    c.fits(n);
    if (!(a.theta > 0)) c.no();
    ocr_axes axes{};
    const bool given = v[12] != Py_None;
    if (given) axes = c.axes(v[12], v[13], n, cache->rot, v[14], v[15]);
    return done(c, [&] { return g_latent_append(ctx, cache, &table, &a, given ? &axes : nullptr); });
OCR_END

// handle, device, cache, table, lens, q, out, scale
OCR_CALL(latent_attend, 8)
    const auto *cache = c.address<const ocr_latent_cache>(v[2]);
    if (!c.ok) return PyLong_FromLong(kOther);
    const ocr_page_table table = c.table(v[3]);
    ocr_latent_decode_args a{};
    int64_t n = table.rows, heads = -1, width = int64_t(cache->rank) + cache->rot, rank = cache->rank;
    int code = 0;
    a.q = c.tokens(v[5], 1u << cache->type, &n, &heads, &width, &a.q_stride, &code);
    a.out = c.tokens(v[6], 1u << cache->type, &n, &heads, &rank, &a.out_stride, &code);
    a.lens = static_cast<const int32_t *>(c.flat(v[4], I32, {n}));
    a.heads = uint32_t(heads), a.scale = float(c.real(v[7]));
    c.fits(heads);
    return done(c, [&] { return g_latent_decode(ctx, cache, &table, &a); });
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

// docs and prefix
template <class A> bool documents(Call &c, PyObject *const *v, A &a, int64_t &ndocs) {
    if (v[0] != Py_None) {
        const at::Tensor *docs = c.tensor(v[0], I32);
        if (!c.ok || docs->dim() != 1 || docs->size(0) < 1 || !docs->is_contiguous()) return false;
        ndocs = docs->size(0) - 1;
        a.docs = static_cast<const int32_t *>(docs->data_ptr());
    }
    a.ndocs = uint32_t(ndocs);
    a.prefix = static_cast<const int32_t *>(c.flat(v[1], I32, {ndocs}, true));
    return true;
}

// handle, device, q, k, v, out, docs, prefix, scale, cap, slopes, weights, window
OCR_CALL(attention, 13)
    ocr_attention_args a{};
    int64_t n = -1, q_heads = -1, kv_heads = -1, dim = -1;
    int code = 0;
    a.q = c.tokens(v[2], HALVES, &n, &q_heads, &dim, &a.q_stride, &a.type);
    a.k = c.tokens(v[3], 1u << a.type, &n, &kv_heads, &dim, &a.k_stride, &code);
    a.v = c.tokens(v[4], 1u << a.type, &n, &kv_heads, &dim, &a.v_stride, &code);
    a.out = c.tokens(v[5], 1u << a.type, &n, &q_heads, &dim, &a.out_stride, &code);
    int64_t ndocs = 1;
    if (!documents(c, v + 6, a, ndocs)) return PyLong_FromLong(kOther);
    a.slopes = static_cast<const float *>(c.flat(v[10], F32, {q_heads}, true));
    a.n = uint32_t(n), a.q_heads = uint32_t(q_heads), a.kv_heads = uint32_t(kv_heads), a.dim = uint32_t(dim);
    a.scale = float(c.real(v[8])), a.cap = float(c.real(v[9]));
    c.fits(n), c.fits(q_heads), c.fits(kv_heads), c.fits(dim), c.fits(ndocs);
    int64_t most = 0;
    float *weights = v[11] == Py_None ? nullptr : static_cast<float *>(c.places(v[11], F32, ndocs, kv_heads, &most));
    const int64_t window = c.whole(v[12]);
    c.fits(window);
    return done(c, [&] { return weights ? g_attention_weights(ctx, &a, weights, uint32_t(most), uint32_t(window)) : g_attention(ctx, &a); });
OCR_END

// handle, device, q, k, r, v, out, docs, prefix, scale
OCR_CALL(latent_attention, 10)
    ocr_latent_attention_args a{};
    int64_t n = -1, heads = -1, width = -1, key = -1, value = -1, ndocs = 1;
    int code = 0;
    a.q = c.tokens(v[2], HALVES, &n, &heads, &width, &a.q_stride, &a.type);
    a.k = c.heads(v[3], 1u << a.type, &n, &heads, &key, &a.k_stride, &a.k_head, &code);
    a.v = c.heads(v[5], 1u << a.type, &n, &heads, &value, &a.v_stride, &a.v_head, &code);
    a.out = c.tokens(v[6], 1u << a.type, &n, &heads, &value, &a.out_stride, &code);
    int64_t rot = width - key;
    if (!c.ok || rot < 0 || (v[4] == Py_None) != (rot == 0)) return PyLong_FromLong(kOther);
    if (rot) a.r = c.rows(v[4], 1u << a.type, &n, &rot, &a.r_stride, &code);
    if (!documents(c, v + 7, a, ndocs)) return PyLong_FromLong(kOther);
    a.n = uint32_t(n), a.heads = uint32_t(heads), a.key = uint32_t(key), a.rot = uint32_t(rot), a.value = uint32_t(value);
    a.scale = float(c.real(v[9]));
    c.fits(n), c.fits(heads), c.fits(width), c.fits(value), c.fits(ndocs);
    return done(c, [&] { return g_latent_attention(ctx, &a); });
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

template <class F> void take(F &f, void *p) { f = reinterpret_cast<F>(p); }
// The functions' addresses, in the order of the pointers above.
PyObject *bind(PyObject *, PyObject *const *v, Py_ssize_t count) {
    constexpr int N = 14;
    if (!count_is(count, N)) return nullptr;
    void *p[N];
    for (int k = 0; k < N; k++)
        if (!(p[k] = PyLong_AsVoidPtr(v[k]))) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no address");
            return nullptr;
        }
    take(g_append, p[0]), take(g_read, p[1]), take(g_attention, p[2]), take(g_decode, p[3]), take(g_beam, p[4]), take(g_fork, p[5]);
    take(g_append_axes, p[6]), take(g_rotate, p[7]), take(g_attention_weights, p[8]), take(g_decode_weights, p[9]), take(g_evict, p[10]);
    take(g_latent_append, p[11]), take(g_latent_decode, p[12]), take(g_latent_attention, p[13]);
    Py_RETURN_NONE;
}

#define OCR_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {OCR_METHOD(bind), OCR_METHOD(append), OCR_METHOD(read), OCR_METHOD(attend), OCR_METHOD(fork),
                         OCR_METHOD(attention), OCR_METHOD(beam_select),
                         OCR_METHOD(append_axes), OCR_METHOD(rotate), OCR_METHOD(evict), OCR_METHOD(latent_append),
                         OCR_METHOD(latent_attend), OCR_METHOD(latent_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
