// The calls of a prompt model's layer (qlinear.fp8_quant_rows and fp8_gemm, prompt.rope and attn) as native code, in the manner of py_states.hpp:
// made in Python they take 13 to 18 us of host time, this way 4 to 6; they answer None for whatever they do not take.
#pragma once

namespace {

// None, or a tensor that is given().  False for anything else.
bool maybe(PyObject* o, const at::Tensor** t) {
    *t = o == Py_None ? nullptr : given(o);
    return o == Py_None || *t;
}
bool real(const at::Tensor& t) { return dt_of(t.scalar_type()) >= 0; }
const void* at_or_null(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
bool vec(const at::Tensor* t, int64_t n) { return !t || (t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == n && t->is_contiguous()); }
PyObject* tuple_of(std::initializer_list<at::Tensor*> ts) {
    PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (at::Tensor* t : ts) {
        PyObject* o = t->defined() ? THPVariable_Wrap(std::move(*t)) : Py_NewRef(Py_None);
        if (!r || !o) {
            Py_XDECREF(o);
            Py_XDECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

// fp8_quant_rows(x, prologue id, norm_w, eps, resid, out) -> (q, scales), (q, scales, sum), or None
PyObject* fp8_quant_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int pro;
    double eps;
    const at::Tensor *x, *w, *resid, *out;
    if (n != 6 || observed() || !small(args[1], &pro) || !number(args[3], &eps)) Py_RETURN_NONE;
    x = given(args[0]);
    if (!x || !maybe(args[2], &w) || !maybe(args[4], &resid) || !maybe(args[5], &out) || !real(*x) || x->dim() != 2 || (x->size(1) > 1 && x->stride(1) != 1)) Py_RETURN_NONE;
    const bool halves = pro == PRO_SWIGLU;
    const int64_t M = x->size(0), K = halves ? x->size(1) / 2 : x->size(1);
    if (M < 1 || K < 1 || (halves && (x->size(1) % 2 || resid)) || (w != nullptr) != (pro == PRO_RMS) || !vec(w, K) || (out && !resid)) Py_RETURN_NONE;
    for (const at::Tensor* t : {resid, out})
        if (t && (t->scalar_type() != x->scalar_type() || t->dim() != 2 || t->size(0) != M || t->size(1) != K || (K > 1 && t->stride(1) != 1))) Py_RETURN_NONE;
    if (out && M > 1 && out->stride(0) < K) Py_RETURN_NONE;
    const auto like = x->options().requires_grad(false);
    at::Tensor q = at::empty({M, K}, like.dtype(at::kFloat8_e4m3fn)), scales = at::empty({(K + 127) / 128, M}, like.dtype(at::kFloat)), total;
    if (resid) total = out ? *out : at::empty({M, K}, like);
    const int rc = without_gil([&] {
        return gpu_fp8_quant_rows(dt_of(x->scalar_type()), pro, x->data_ptr(), x->stride(0), at_or_null(resid), resid ? resid->stride(0) : 0, memory(total), resid ? total.stride(0) : 0, K,
                                  (const float*)at_or_null(w), (float)eps, q.data_ptr(), (float*)scales.data_ptr(), M, int_of(M), int_of(K), stream_now());
    });
    if (rc != 0) Py_RETURN_NONE;
    return resid ? tuple_of({&q, &scales, &total}) : tuple_of({&q, &scales});
    END_HANDLE_TH_ERRORS
}

// fp8_gemm(A, W, xs, ws, bias, out_dtype, D) -> D, or None
PyObject* fp8_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const at::Tensor *bias, *given_d;
    if (n != 7 || observed() || !THPDtype_Check(args[5])) Py_RETURN_NONE;
    const at::ScalarType type = ((THPDtype*)args[5])->scalar_type;
    const at::Tensor *A = given(args[0]), *W = given(args[1]), *xs = given(args[2]), *ws = given(args[3]);
    if (!A || !W || !xs || !ws || !maybe(args[4], &bias) || !maybe(args[6], &given_d) || dt_of(type) < 0) Py_RETURN_NONE;
    if (!dense(*A, at::kFloat8_e4m3fn) || !dense(*W, at::kFloat8_e4m3fn) || A->dim() != 2 || W->dim() != 2 || A->size(1) != W->size(1) || !dense(*ws, at::kFloat) || xs->scalar_type() != at::kFloat) Py_RETURN_NONE;
    const int64_t M = A->size(0), K = A->size(1), N = W->size(0), G = (K + 127) / 128;
    if (M < 1 || N < 1 || K < 1 || xs->dim() != 2 || xs->size(0) != G || xs->size(1) != M || (M > 1 && xs->stride(1) != 1) || (G > 1 && xs->stride(0) < M) || ws->dim() != 2 || ws->size(0) != (N + 127) / 128 || ws->size(1) != G) Py_RETURN_NONE;
    if (bias && (!dense(*bias, type) || bias->dim() != 1 || bias->size(0) != N)) Py_RETURN_NONE;
    if (given_d && (!dense(*given_d, type) || given_d->dim() != 2 || given_d->size(0) != M || given_d->size(1) != N)) Py_RETURN_NONE;
    at::Tensor D = given_d ? *given_d : at::empty({M, N}, A->options().dtype(type).requires_grad(false));
    const int64_t stride = G > 1 ? xs->stride(0) : M;
    at::Tensor work = scratch_of(gpu_fp8_gemm_workspace(M, N, K, dt_of(type)), *A);
    const int rc = without_gil([&] {
        return gpu_fp8_gemm(A->data_ptr(), W->data_ptr(), (const float*)xs->data_ptr(), stride, (const float*)ws->data_ptr(), at_or_null(bias), D.data_ptr(), memory(work), M, N, K, dt_of(type),
                            stream_now());
    });
    if (rc == 0) return THPVariable_Wrap(std::move(D));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

bool token_heads(const at::Tensor& t, int64_t tokens, int64_t dim, at::ScalarType type) {
    return t.scalar_type() == type && t.dim() == 3 && t.size(0) == tokens && t.size(2) == dim && t.stride(2) == 1;
}

// rope(q, k, positions, freqs, interleaved, factor, q_norm, k_norm, eps) -> (q, k), or None
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    double factor, eps;
    const at::Tensor *k, *qn, *kn;
    if (n != 9 || observed() || !PyBool_Check(args[4]) || !number(args[5], &factor) || !number(args[8], &eps)) Py_RETURN_NONE;
    const at::Tensor *q = given(args[0]), *positions = given(args[2]), *freqs = given(args[3]);
    if (!q || !positions || !freqs || !maybe(args[1], &k) || !maybe(args[6], &qn) || !maybe(args[7], &kn) || !real(*q) || q->dim() != 3 || (k && k->dim() != 3)) Py_RETURN_NONE;
    const int64_t T = q->size(0), h = q->size(1), d = q->size(2), hk = k ? k->size(1) : 0;
    if (T < 1 || d < 1 || !token_heads(*q, T, d, q->scalar_type()) || (k && !token_heads(*k, T, d, q->scalar_type())) || !ints(positions, 1) || positions->size(0) != T || !vec(qn, d) || !vec(kn, d) ||
        freqs->scalar_type() != at::kDouble || freqs->dim() != 1 || !freqs->is_contiguous()) Py_RETURN_NONE;
    const auto like = q->options().requires_grad(false);
    at::Tensor qo = at::empty({T, h, d}, like), ko;
    if (k) ko = at::empty({T, hk, d}, like);
    const int rc = without_gil([&] {
        return gpu_rope(dt_of(q->scalar_type()), q->data_ptr(), q->stride(0), q->stride(1), qo.data_ptr(), qo.stride(0), qo.stride(1), int_of(h), at_or_null(k), k ? k->stride(0) : 0, k ? k->stride(1) : 0,
                        memory(ko), k ? ko.stride(0) : 0, k ? ko.stride(1) : 0, int_of(hk), (const int32_t*)positions->data_ptr(), (const double*)freqs->data_ptr(), int_of(2 * freqs->size(0)),
                        args[4] == Py_True, (float)factor, (const float*)at_or_null(qn), (const float*)at_or_null(kn), (float)eps, int_of(T), int_of(d), stream_now());
    });
    if (rc != 0) Py_RETURN_NONE;
    return tuple_of({&qo, &ko});
    END_HANDLE_TH_ERRORS
}

// prompt_attn(q, k, v, starts, scale, causal) -> tensor, or None
PyObject* prompt_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    double scale;
    if (n != 6 || observed() || !number(args[4], &scale) || !PyBool_Check(args[5])) Py_RETURN_NONE;
    const at::Tensor *q = given(args[0]), *k = given(args[1]), *v = given(args[2]), *starts = given(args[3]);
    if (!q || !k || !v || !ints(starts, 1) || starts->size(0) < 1 || !half_type(*q) || q->dim() != 3 || k->dim() != 3) Py_RETURN_NONE;
    const int64_t T = q->size(0), h = q->size(1), d = q->size(2), hk = k->size(1);
    if (T < 1 || hk < 1 || h < 1 || h % hk != 0 || !token_heads(*q, T, d, q->scalar_type()) || !token_heads(*k, T, d, q->scalar_type()) || !token_heads(*v, T, d, q->scalar_type()) || v->size(1) != hk) Py_RETURN_NONE;
    const int it = int_of(T), ih = int_of(h), ihk = int_of(hk), id = int_of(d), in = int_of(starts->size(0) - 1);
    at::Tensor o = at::empty({T, h, d}, q->options().requires_grad(false));
    const int rc = without_gil([&] {
        return gpu_prompt_attn(dt_of(q->scalar_type()), q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), o.data_ptr(),
                               o.stride(0), o.stride(1), (const int32_t*)starts->data_ptr(), in, it, ih, ihk, id, (float)scale, args[5] == Py_True, stream_now());
    });
    if (rc == 0) return THPVariable_Wrap(std::move(o));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

}  // namespace
