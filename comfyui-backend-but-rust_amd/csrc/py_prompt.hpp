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

// The runs of bytes that a tensor has, as _runs in qlinear.py finds them: up to two steps between them, the wider one last.
struct Runs {
    int64_t at, width, n[2] = {1, 1}, step[2] = {0, 0};
    int axes = 0;
    explicit Runs(const at::Tensor& t) : at((int64_t)(uintptr_t)t.data_ptr()), width((int64_t)t.element_size()) {
        int64_t s[3], c[3];
        int dims = 0;
        for (int64_t i = t.dim() - 1; i >= 0; --i) {      // (by their steps: three at most)
            if (t.size(i) == 1) continue;
            int j = dims++;
            for (; j > 0 && s[j - 1] > t.stride(i) * width; --j) s[j] = s[j - 1], c[j] = c[j - 1];
            s[j] = t.stride(i) * width, c[j] = t.size(i);
        }
        for (int i = 0; i < dims; ++i) {
            if (axes == 0 && s[i] <= width) width += (c[i] - 1) * s[i];
            else if (axes && s[i] == n[axes - 1] * step[axes - 1]) n[axes - 1] *= c[i];
            else if (axes < 2) n[axes] = c[i], step[axes++] = s[i];
        }
    }
    int64_t reach(int upto) const {
        int64_t r = width;
        for (int i = 0; i < upto; ++i) r += (n[i] - 1) * step[i];
        return r;
    }
};
// Whether an output of up to three axes may share memory with another tensor: where this is not clear from their ranges and from what they have of the steps
// between their rows, Python looks (qlinear._meet).
bool may_meet(const at::Tensor& out, const at::Tensor* t) {
    if (!t || !out.numel() || !t->numel()) return false;
    if (out.dim() > 3 || t->dim() > 3) return true;
    const Runs a(out), b(*t);
    if (a.at + a.reach(a.axes) <= b.at || b.at + b.reach(b.axes) <= a.at) return false;
    if (a.axes + b.axes == 0) return true;
    const auto clear = [&](int64_t step, int64_t first, int64_t second) {
        const int64_t r = ((b.at - a.at) % step + step) % step;
        return first <= r && r + second <= step;
    };
    int64_t g = 0;
    for (int i = 0; i < a.axes; ++i) g = std::gcd(g, a.step[i]);
    for (int i = 0; i < b.axes; ++i) g = std::gcd(g, b.step[i]);
    if (clear(g, a.width, b.width)) return false;
    return !(a.axes && b.axes && a.step[a.axes - 1] == b.step[b.axes - 1] && clear(a.step[a.axes - 1], a.reach(a.axes - 1), b.reach(b.axes - 1)));
}
bool in_place_of(const at::Tensor& out, const at::Tensor& t) {
    if (out.data_ptr() != t.data_ptr() || out.sizes() != t.sizes() || out.scalar_type() != t.scalar_type()) return false;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) != 1 && t.stride(i) != out.stride(i)) return false;
    return true;
}
// The rows of an output lie apart from each other, as qlinear._apart has it, and from what is read, unless it goes in the place of one of `places`.
bool separate(const at::Tensor& out, std::initializer_list<const at::Tensor*> reads, std::initializer_list<const at::Tensor*> places = {}) {
    if (out.dim() > 3) return false;
    const Runs a(out);
    if (out.numel() && a.width < out.size(-1) * (int64_t)out.element_size()) return false;
    int64_t bytes = out.numel() * (int64_t)out.element_size();
    if (out.numel() && (a.axes == 0 ? a.width != bytes : a.step[0] < a.width || a.n[0] * (a.axes > 1 ? a.n[1] : 1) * a.width != bytes || (a.axes > 1 && a.step[1] < a.reach(1)))) return false;
    for (const at::Tensor* t : places)
        if (t && !in_place_of(out, *t) && may_meet(out, t)) return false;
    for (const at::Tensor* t : reads)
        if (may_meet(out, t)) return false;
    return true;
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
    if (out && !separate(*out, {w}, {x, resid})) Py_RETURN_NONE;
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
    if (given_d && !separate(*given_d, {A, W, xs, ws, bias})) Py_RETURN_NONE;
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

// rope(q, k, positions, freqs, interleaved, factor, q_norm, k_norm, eps, out) -> (q, k), or None
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    double factor, eps;
    const at::Tensor *k, *qn, *kn, *q_to = nullptr, *k_to = nullptr;
    if (n != 10 || observed() || !PyBool_Check(args[4]) || !number(args[5], &factor) || !number(args[8], &eps)) Py_RETURN_NONE;
    const at::Tensor *q = given(args[0]), *positions = given(args[2]), *freqs = given(args[3]);
    if (!q || !positions || !freqs || !maybe(args[1], &k) || !maybe(args[6], &qn) || !maybe(args[7], &kn) || !real(*q) || q->dim() != 3 || (k && k->dim() != 3)) Py_RETURN_NONE;
    const int64_t T = q->size(0), h = q->size(1), d = q->size(2), hk = k ? k->size(1) : 0;
    if (T < 1 || d < 1 || !token_heads(*q, T, d, q->scalar_type()) || (k && !token_heads(*k, T, d, q->scalar_type())) || !ints(positions, 1) || positions->size(0) != T || !vec(qn, d) || !vec(kn, d) ||
        freqs->scalar_type() != at::kDouble || freqs->dim() != 1 || !freqs->is_contiguous()) Py_RETURN_NONE;
    const auto like = q->options().requires_grad(false);
    if (args[9] != Py_None) {
        if (!PyTuple_Check(args[9]) || PyTuple_GET_SIZE(args[9]) != 2 || !maybe(PyTuple_GET_ITEM(args[9], 0), &q_to) || !maybe(PyTuple_GET_ITEM(args[9], 1), &k_to) || !q_to || !k != !k_to) Py_RETURN_NONE;
        if (!token_heads(*q_to, T, d, q->scalar_type()) || q_to->size(1) != h || !separate(*q_to, {k, positions, freqs, qn, kn}, {q})) Py_RETURN_NONE;
        if (k && (!token_heads(*k_to, T, d, q->scalar_type()) || k_to->size(1) != hk || !separate(*k_to, {q_to, q, positions, freqs, qn, kn}, {k}))) Py_RETURN_NONE;
    }
    at::Tensor qo = q_to ? *q_to : at::empty({T, h, d}, like), ko;
    if (k) ko = k_to ? *k_to : at::empty({T, hk, d}, like);
    const int rc = without_gil([&] {
        return gpu_rope(dt_of(q->scalar_type()), q->data_ptr(), q->stride(0), q->stride(1), qo.data_ptr(), qo.stride(0), qo.stride(1), int_of(h), at_or_null(k), k ? k->stride(0) : 0, k ? k->stride(1) : 0,
                        memory(ko), k ? ko.stride(0) : 0, k ? ko.stride(1) : 0, int_of(hk), (const int32_t*)positions->data_ptr(), (const double*)freqs->data_ptr(), int_of(2 * freqs->size(0)),
                        args[4] == Py_True, (float)factor, (const float*)at_or_null(qn), (const float*)at_or_null(kn), (float)eps, int_of(T), int_of(d), stream_now());
    });
    if (rc != 0) Py_RETURN_NONE;
    return tuple_of({&qo, &ko});
    END_HANDLE_TH_ERRORS
}

// prompt_attn(q, k, v, starts, scale, causal, out) -> tensor, or None
PyObject* prompt_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    double scale;
    const at::Tensor* to;
    if (n != 7 || observed() || !maybe(args[6], &to) || !number(args[4], &scale) || !PyBool_Check(args[5])) Py_RETURN_NONE;
    const at::Tensor *q = given(args[0]), *k = given(args[1]), *v = given(args[2]), *starts = given(args[3]);
    if (!q || !k || !v || !ints(starts, 1) || starts->size(0) < 1 || !half_type(*q) || q->dim() != 3 || k->dim() != 3) Py_RETURN_NONE;
    const int64_t T = q->size(0), h = q->size(1), d = q->size(2), hk = k->size(1);
    if (T < 1 || hk < 1 || h < 1 || h % hk != 0 || !token_heads(*q, T, d, q->scalar_type()) || !token_heads(*k, T, d, q->scalar_type()) || !token_heads(*v, T, d, q->scalar_type()) || v->size(1) != hk) Py_RETURN_NONE;
    const int it = int_of(T), ih = int_of(h), ihk = int_of(hk), id = int_of(d), in = int_of(starts->size(0) - 1);
    if (to && (!token_heads(*to, T, d, q->scalar_type()) || to->size(1) != h || !separate(*to, {k, v, starts}, {q}))) Py_RETURN_NONE;
    at::Tensor o = to ? *to : at::empty({T, h, d}, q->options().requires_grad(false));
    const int rc = without_gil([&] {
        return gpu_prompt_attn(dt_of(q->scalar_type()), q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), o.data_ptr(),
                               o.stride(0), o.stride(1), (const int32_t*)starts->data_ptr(), in, it, ih, ihk, id, (float)scale, args[5] == Py_True, stream_now());
    });
    if (rc == 0) return THPVariable_Wrap(std::move(o));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

}  // namespace
