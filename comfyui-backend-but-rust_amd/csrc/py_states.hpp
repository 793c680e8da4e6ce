// qlinear.cross_attn and kvcache's calls as native code, for csrc/py_linear.cpp: checks, allocation and launch behind one call from Python.
// Made in Python a call takes 12 to 16 us of host time, more than a token's attention takes on the GPU; this way 3 to 5.  They answer None
// for whatever they do not take, and the caller then does the whole call in Python, which raises what there is to raise.
#pragma once

namespace {

// A tensor whose memory a kernel may read: on the current device, without a gradient to record or a tangent to carry on.
const at::Tensor* given(PyObject* o) {
    const at::Tensor* t = plain(o);
    if (!t || !t->is_cuda() || t->layout() != at::kStrided || t->device().index() != c10::hip::current_device()) return nullptr;
    if (!t->unsafeGetTensorImpl()->autograd_meta()) return t;      // which both would be part of
    if (t->requires_grad() && at::GradMode::is_enabled()) return nullptr;
    return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined() ? nullptr : t;
}
bool ints(const at::Tensor* t, int64_t dims) { return t && t->scalar_type() == at::kInt && t->dim() == dims && t->is_contiguous(); }
bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
bool number(PyObject* o, double* out) {
    if (!PyFloat_CheckExact(o)) return false;
    *out = PyFloat_AS_DOUBLE(o);
    return true;
}
bool small(PyObject* o, int* out) {
    if (!PyLong_CheckExact(o)) return false;
    int over = 0;
    const long v = PyLong_AsLongAndOverflow(o, &over);
    if (over || v < 0 || v > 0x7fffffff) return false;
    *out = (int)v;
    return true;
}
int int_of(int64_t v) { return v > 0x7fffffff ? -1 : (int)v; }      // refused by the launcher
void* stream_now() { return (void*)c10::hip::getCurrentHIPStream().stream(); }
at::Tensor scratch_of(int64_t bytes, const at::Tensor& like) { return bytes ? at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false)) : at::Tensor(); }
void* memory(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <class Call> int without_gil(Call call) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = call();
    Py_END_ALLOW_THREADS
    return rc;
}

// (k, v, k_scale, v_scale) of one layer
struct CacheOf {
    const at::Tensor *k, *v, *ks, *vs;
    int pages, heads, page, dim;
    bool take(PyObject* const* a, int64_t dims) {
        k = given(a[0]), v = given(a[1]), ks = given(a[2]), vs = given(a[3]);
        if (!k || !v || !ks || !vs || k->scalar_type() != at::kChar || v->scalar_type() != at::kChar || k->dim() != dims || !k->is_contiguous() || !v->is_contiguous() ||
            v->sizes() != k->sizes() || ks->scalar_type() != at::kFloat || vs->scalar_type() != at::kFloat || !ks->is_contiguous() || !vs->is_contiguous() || vs->sizes() != ks->sizes())
            return false;
        const auto s = k->sizes();
        if (ks->dim() != dims - 1 || s[dims - 2] % 16 != 0 || ks->size(dims - 2) != s[dims - 2] / 16) return false;
        for (int64_t i = 0; i < dims - 2; ++i)
            if (ks->size(i) != s[i]) return false;
        pages = int_of(s[dims - 4]), heads = int_of(s[dims - 3]), page = int_of(s[dims - 2]), dim = int_of(s[dims - 1]);
        return true;
    }
};
// (starts, lens, table, most)
struct RowsOf {
    const at::Tensor *starts, *lens, *table;
    int n, cols, most;
    bool take(PyObject* const* a) {
        starts = given(a[0]), lens = given(a[1]), table = given(a[2]);
        if (!ints(starts, 1) || !ints(lens, 1) || !ints(table, 2) || starts->size(0) != lens->size(0) + 1 || table->size(0) != lens->size(0) || !small(a[3], &most)) return false;
        n = int_of(lens->size(0)), cols = int_of(table->size(1));
        return true;
    }
};
bool heads_of(const at::Tensor* t, int64_t heads, int64_t dim) {
    return t && half_type(*t) && t->dim() == 3 && (heads < 0 || t->size(1) == heads) && t->size(2) == dim && t->stride(2) == 1;
}

// cross_attn(q, k, v, scale, k_lens, mask) -> tensor, or None
PyObject* cross_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    double scale;
    if (n != 6 || observed() || !number(args[3], &scale)) Py_RETURN_NONE;
    const at::Tensor *q = given(args[0]), *k = given(args[1]), *v = given(args[2]), *lens = args[4] == Py_None ? nullptr : given(args[4]), *mask = args[5] == Py_None ? nullptr : given(args[5]);
    if (!q || !k || !v || (args[4] != Py_None && !lens) || (args[5] != Py_None && !mask) || !half_type(*q) || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type()) Py_RETURN_NONE;
    if (q->dim() != 4 || k->dim() != 4 || v->sizes() != k->sizes() || q->stride(3) != 1 || k->stride(3) != 1 || v->stride(3) != 1) Py_RETURN_NONE;
    const int64_t b = q->size(0), lq = q->size(1), h = q->size(2), d = q->size(3), lk = k->size(1), hk = k->size(2);
    if (k->size(0) != b || k->size(3) != d || hk < 1 || h < 1 || h % hk != 0 || b < 1 || lq < 1 || lk < 1) Py_RETURN_NONE;
    if (lens && (!ints(lens, 1) || lens->size(0) != b)) Py_RETURN_NONE;
    if (mask && ((mask->scalar_type() != at::kBool && mask->scalar_type() != at::kFloat) || mask->dim() < 1 || mask->dim() > 2 || mask->size(-1) != lk ||
                 (mask->dim() == 2 && mask->size(0) != b) || (lk > 1 && mask->stride(-1) != 1))) Py_RETURN_NONE;
    const int ib = int_of(b), ilq = int_of(lq), ilk = int_of(lk), ih = int_of(h), ihk = int_of(hk), id = int_of(d);
    at::Tensor o = at::empty({b, lq, h, d}, q->options().requires_grad(false)), ws = scratch_of(gpu_cross_attn_workspace(ib, ilq, ilk, ih, ihk, id), *q);
    const int rc = without_gil([&] {
        return gpu_cross_attn(dt_of(q->scalar_type()), q->data_ptr(), k->data_ptr(), v->data_ptr(), o.data_ptr(), memory(ws), ib, ilq, ilk, ih, ihk, id, q->stride(0), q->stride(1),
                              q->stride(2), k->stride(0), k->stride(1), k->stride(2), v->stride(0), v->stride(1), v->stride(2), o.stride(0), o.stride(1), o.stride(2), (float)scale,
                              lens ? (const int32_t*)lens->data_ptr() : nullptr, mask ? mask->data_ptr() : nullptr, !mask ? 0 : mask->scalar_type() == at::kBool ? 1 : 2,
                              mask && mask->dim() == 2 ? mask->stride(0) : 0, stream_now());
    });
    if (rc == 0) return THPVariable_Wrap(std::move(o));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// kv8_attn(q, k, v, k_scale, v_scale, starts, lens, table, most, scale, causal) -> tensor, or None
PyObject* kv8_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    double scale;
    CacheOf c;
    RowsOf r;
    if (n != 11 || observed() || !number(args[9], &scale) || !PyBool_Check(args[10]) || !c.take(args + 1, 4) || !r.take(args + 5)) Py_RETURN_NONE;
    const at::Tensor* q = given(args[0]);
    if (!heads_of(q, -1, c.dim) || q->size(1) < 1 || c.heads < 1 || q->size(1) % c.heads != 0) Py_RETURN_NONE;
    const int h = int_of(q->size(1)), rows = int_of(q->size(0));
    at::Tensor o = at::empty(q->sizes(), q->options().requires_grad(false)), ws = scratch_of(gpu_kv8_attn_workspace(r.n, r.most, h, c.heads, c.dim, c.page, r.cols), *q);
    const int rc = without_gil([&] {
        return gpu_kv8_attn(dt_of(q->scalar_type()), q->data_ptr(), q->stride(0), q->stride(1), o.data_ptr(), o.stride(0), o.stride(1), memory(ws), (const int8_t*)c.k->data_ptr(),
                            (const int8_t*)c.v->data_ptr(), (const float*)c.ks->data_ptr(), (const float*)c.vs->data_ptr(), c.pages, c.page, (const int32_t*)r.starts->data_ptr(),
                            (const int32_t*)r.lens->data_ptr(), (const int32_t*)r.table->data_ptr(), r.cols, r.n, rows, r.most, h, c.heads, c.dim, (float)scale, args[10] == Py_True,
                            stream_now());
    });
    if (rc == 0) return THPVariable_Wrap(std::move(o));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// kv8_store(k, v, cache k, v, k_scale, v_scale, starts, lens, table, most) -> True, or None
PyObject* kv8_store(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    CacheOf c;
    RowsOf r;
    if (n != 10 || observed() || !c.take(args + 2, 4) || !r.take(args + 6)) Py_RETURN_NONE;
    const at::Tensor *k = given(args[0]), *v = given(args[1]);
    if (!heads_of(k, c.heads, c.dim) || !heads_of(v, c.heads, c.dim) || v->size(0) != k->size(0) || v->scalar_type() != k->scalar_type()) Py_RETURN_NONE;
    const int rc = without_gil([&] {
        return gpu_kv8_store(dt_of(k->scalar_type()), k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), (int8_t*)c.k->data_ptr(),
                             (int8_t*)c.v->data_ptr(), (float*)c.ks->data_ptr(), (float*)c.vs->data_ptr(), c.pages, c.page, (const int32_t*)r.starts->data_ptr(),
                             (const int32_t*)r.lens->data_ptr(), (const int32_t*)r.table->data_ptr(), r.cols, r.n, int_of(k->size(0)), r.most, c.heads, c.dim, stream_now());
    });
    if (rc == 0) Py_RETURN_TRUE;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// kv8_read(cache k, v, k_scale, v_scale, starts, lens, table, most, tokens, dtype) -> (k, v), or None
PyObject* kv8_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    CacheOf c;
    RowsOf r;
    int tokens;
    if (n != 10 || observed() || !c.take(args, 4) || !r.take(args + 4) || !small(args[8], &tokens) || !THPDtype_Check(args[9])) Py_RETURN_NONE;
    const at::ScalarType type = ((THPDtype*)args[9])->scalar_type;
    if (dt_of(type) < 0) Py_RETURN_NONE;
    at::Tensor out[2];
    for (at::Tensor& t : out) t = at::empty({tokens, c.heads, c.dim}, c.k->options().dtype(type).requires_grad(false));
    const int rc = without_gil([&] {
        return gpu_kv8_read(dt_of(type), out[0].data_ptr(), out[0].stride(0), out[0].stride(1), out[1].data_ptr(), out[1].stride(0), out[1].stride(1), (const int8_t*)c.k->data_ptr(),
                            (const int8_t*)c.v->data_ptr(), (const float*)c.ks->data_ptr(), (const float*)c.vs->data_ptr(), c.pages, c.page, (const int32_t*)r.starts->data_ptr(),
                            (const int32_t*)r.lens->data_ptr(), (const int32_t*)r.table->data_ptr(), r.cols, r.n, tokens, r.most, c.heads, c.dim, stream_now());
    });
    if (rc != 0) Py_RETURN_NONE;
    PyObject *k = THPVariable_Wrap(std::move(out[0])), *v = k ? THPVariable_Wrap(std::move(out[1])) : nullptr, *pair = v ? PyTuple_Pack(2, k, v) : nullptr;
    Py_XDECREF(k);
    Py_XDECREF(v);
    return pair;
    END_HANDLE_TH_ERRORS
}

// kv8_copy_pages(cache k, v, k_scale, v_scale, src, dst) -> True, or None
PyObject* kv8_copy_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    CacheOf c;
    if (n != 6 || observed()) Py_RETURN_NONE;
    const at::Tensor *k = given(args[0]), *src = given(args[4]), *dst = given(args[5]);
    if (!k || (k->dim() != 4 && k->dim() != 5) || !c.take(args, k->dim()) || !ints(src, 1) || !ints(dst, 1) || src->size(0) != dst->size(0)) Py_RETURN_NONE;
    const int rc = without_gil([&] {
        return gpu_kv8_copy_pages((int8_t*)c.k->data_ptr(), (int8_t*)c.v->data_ptr(), (float*)c.ks->data_ptr(), (float*)c.vs->data_ptr(), c.k->dim() == 5 ? int_of(c.k->size(0)) : 1, c.pages,
                                  c.page, c.heads, c.dim, (const int32_t*)src->data_ptr(), (const int32_t*)dst->data_ptr(), int_of(src->size(0)), stream_now());
    });
    if (rc == 0) Py_RETURN_TRUE;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

}  // namespace
