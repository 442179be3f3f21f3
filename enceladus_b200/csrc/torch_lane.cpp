// The short way from Python to the decoding step's entry points for torch tensors.
//
// The kernels of a decoding step run for a few microseconds, and ops.py spends more than that on reading shapes, strides and
// addresses of up to eleven tensors one attribute at a time (12 us a call, 46 with the launch path).  The functions here read them where torch keeps
// them, check the same things and make the same call into libenc_b200.so (3.6 us for append_kv).  They decide nothing: whatever is not a call that
// can go straight through - an argument that is wrong, NumPy arrays, another device, a zero-sized launch - is answered with
// NotImplemented, and ops.py goes its general way, which also words the errors.  A status other than ENC_OK is returned as an
// int for ops.py to raise.  Functions of libenc_b200.so are reached through addresses given once by init(), so nothing is linked
// here but torch, which the process has loaded already.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdlib>

#include "../../include/enceladus_b200.h"

namespace {

decltype(&enc_append_kv) append_fn = nullptr;
decltype(&enc_paged_attention) attention_fn = nullptr;
decltype(&enc_paged_attention_work_bytes) work_fn = nullptr;
decltype(&enc_penalize_logits) logits_fn = nullptr;

PyObject *not_here() { return Py_NewRef(Py_NotImplemented); }

// What all tensors of a launch have to be: plain strided CUDA tensors on the current device.
struct Launch {
    int device = -1;  // asked for at the first CUDA tensor: without one there may be no driver
    bool ok = attention_fn != nullptr && getenv("ENCELADUS_INTERPRET") == nullptr;

    const at::Tensor *tensor(PyObject *o) {  // nullptr for None
        if (o == Py_None) return nullptr;
        if (!THPVariable_CheckExact(o)) {
            ok = false;
            return nullptr;
        }
        const at::Tensor &t = THPVariable_Unpack(o);
        ok = ok && t.is_cuda() && t.layout() == at::kStrided;
        if (ok && device < 0) device = c10::cuda::current_device();
        ok = ok && t.get_device() == device;
        return &t;
    }
    const at::Tensor *needed(PyObject *o) {
        const at::Tensor *t = tensor(o);
        ok = ok && t;
        return t;
    }
    void *stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
};

int dtype_code(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return ENC_F32;
        case at::kHalf: return ENC_F16;
        case at::kBFloat16: return ENC_BF16;
        default: return -1;
    }
}
bool is(const at::Tensor *t, at::ScalarType s) { return !t || t->scalar_type() == s; }
bool contiguous_rows(const at::Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }
bool writable(const at::Tensor &t) {  // no two elements share memory through a stride of zero
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.stride(i) == 0 && t.size(i) > 1) return false;
    return true;
}
bool heads(const at::Tensor &t, int64_t rows, int64_t n, int64_t head_dim, int code) {
    return t.dim() == 3 && t.size(0) == rows && t.size(1) == n && t.size(2) == head_dim && contiguous_rows(t) && dtype_code(t) == code;
}
bool row(const at::Tensor *t, int64_t n, at::ScalarType s) {
    return t && t->dim() == 1 && t->size(0) == n && (n <= 1 || t->stride(0) == 1) && t->scalar_type() == s;
}
bool rows(const at::Tensor *t, int64_t n, at::ScalarType s) { return t && t->dim() == 2 && t->size(0) == n && contiguous_rows(*t) && t->scalar_type() == s; }
template <typename T> T *ptr(const at::Tensor *t) { return t ? reinterpret_cast<T *>(t->data_ptr()) : nullptr; }

bool fill_cache(enc_paged_cache &c, const at::Tensor &k, const at::Tensor &v, const at::Tensor &table, int code) {
    if (k.dim() != 4 || k.sizes() != v.sizes() || table.dim() != 2 || k.numel() == 0 || table.numel() == 0) return false;
    if (!contiguous_rows(k) || !contiguous_rows(v) || !contiguous_rows(table)) return false;
    if (dtype_code(k) != code || dtype_code(v) != code || table.scalar_type() != at::kInt) return false;
    c = {k.data_ptr(), v.data_ptr(), reinterpret_cast<const int32_t *>(table.data_ptr()), k.size(0), k.size(2), k.size(1), k.size(3), table.size(0),
         table.size(1), table.stride(0), k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2)};
    return true;
}

// (k, v, k_cache, v_cache, block_table, seq_ids, positions, cos, sin, q, q_out, interleaved) -> q_out
PyObject *append_kv(PyObject *, PyObject *const *x, Py_ssize_t n) {
    if (n != 12) return not_here();
    try {
        Launch at;
        const at::Tensor *k = at.needed(x[0]), *v = at.needed(x[1]), *kc = at.needed(x[2]), *vc = at.needed(x[3]), *table = at.needed(x[4]);
        const at::Tensor *ids = at.needed(x[5]), *pos = at.needed(x[6]), *cos = at.tensor(x[7]), *sin = at.tensor(x[8]);
        const at::Tensor *q = at.tensor(x[9]), *out = at.tensor(x[10]);
        const int interleaved = PyObject_IsTrue(x[11]);
        if (!at.ok || interleaved < 0 || (cos == nullptr) != (sin == nullptr) || (out && !q) || k->dim() != 3) {
            PyErr_Clear();
            return not_here();
        }
        const int code = dtype_code(*k);
        const int64_t tokens = k->size(0);
        enc_paged_cache cache;
        if (code < 0 || tokens == 0 || !fill_cache(cache, *kc, *vc, *table, code) || !writable(*kc) || !writable(*vc)) return not_here();
        const int64_t d = cache.head_dim;
        if (!heads(*k, tokens, cache.kv_heads, d, code) || !heads(*v, tokens, cache.kv_heads, d, code) || !row(ids, tokens, at::kInt) ||
            !row(pos, tokens, at::kInt))
            return not_here();
        enc_append_args g = {};
        g.k = k->data_ptr(); g.v = v->data_ptr(); g.seq_ids = ptr<int32_t>(ids); g.positions = ptr<int32_t>(pos);
        g.tokens = tokens; g.interleaved = interleaved;
        g.k_stride_token = k->stride(0); g.k_stride_head = k->stride(1); g.v_stride_token = v->stride(0); g.v_stride_head = v->stride(1);
        if (cos) {
            if (cos->dim() != 2 || cos->sizes() != sin->sizes() || cos->strides() != sin->strides() || !contiguous_rows(*cos) ||
                !is(cos, at::kFloat) || !is(sin, at::kFloat) || 2 * cos->size(1) > d || cos->numel() == 0)
                return not_here();
            g.cos = ptr<float>(cos); g.sin = ptr<float>(sin);
            g.rot_dim = 2 * cos->size(1); g.num_positions = cos->size(0); g.stride_cos = cos->stride(0);
        }
        at::Tensor made;
        if (q) {
            if (q->dim() != 3 || q->size(1) == 0 || !heads(*q, tokens, q->size(1), d, code)) return not_here();
            if (out) {
                if (!heads(*out, tokens, q->size(1), d, code) || !writable(*out)) return not_here();
            } else {
                made = at::empty(q->sizes(), q->options());
                out = &made;
            }
            g.q = q->data_ptr(); g.q_out = out->data_ptr(); g.q_heads = q->size(1);
            g.q_stride_token = q->stride(0); g.q_stride_head = q->stride(1); g.o_stride_token = out->stride(0); g.o_stride_head = out->stride(1);
        }
        int status;
        void *stream = at.stream();
        Py_BEGIN_ALLOW_THREADS
        status = append_fn(&cache, &g, code, ENC_VARIANT_AUTO, stream);
        Py_END_ALLOW_THREADS
        if (status != ENC_OK) return PyLong_FromLong(status);
        if (!q) Py_RETURN_NONE;
        return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(x[10]);
    } catch (...) {
        PyErr_Clear();
        return not_here();
    }
}

// (q, k_cache, v_cache, block_table, seq_lens, sm_scale, window, o, return_lse) -> o or (o, lse)
PyObject *paged_attention(PyObject *, PyObject *const *x, Py_ssize_t n) {
    if (n != 9) return not_here();
    try {
        Launch at;
        const at::Tensor *q = at.needed(x[0]), *kc = at.needed(x[1]), *vc = at.needed(x[2]), *table = at.needed(x[3]), *lens = at.needed(x[4]);
        const at::Tensor *o = at.tensor(x[7]);
        const double scale = x[5] == Py_None ? 0.0 : PyFloat_AsDouble(x[5]);
        const long long window = PyLong_AsLongLong(x[6]);
        const int return_lse = PyObject_IsTrue(x[8]);
        if (!at.ok || PyErr_Occurred() || window < 0 || return_lse < 0 || q->dim() != 3) {
            PyErr_Clear();
            return not_here();
        }
        const int code = dtype_code(*q);
        const int64_t seqs = q->size(0), q_heads = q->size(1);
        enc_paged_cache cache;
        if (code < 0 || seqs == 0 || !fill_cache(cache, *kc, *vc, *table, code) || cache.num_seqs != seqs || q_heads == 0 || q_heads % cache.kv_heads ||
            cache.head_dim > 256 || !heads(*q, seqs, q_heads, cache.head_dim, code) || !row(lens, seqs, at::kInt))
            return not_here();
        at::Tensor made, lse, work;
        if (o) {
            if (!heads(*o, seqs, q_heads, cache.head_dim, code) || !writable(*o)) return not_here();
        } else {
            made = at::empty(q->sizes(), q->options());
            o = &made;
        }
        enc_paged_attention_args g = {};
        g.work_bytes = work_fn(&cache, q_heads, code, ENC_VARIANT_AUTO);
        if (g.work_bytes < 0) return not_here();
        if (g.work_bytes > 0) {  // from torch's caching allocator on this stream: nothing is shared with other launches
            work = at::empty({g.work_bytes}, q->options().dtype(at::kByte));
            g.work = work.data_ptr();
        }
        if (return_lse) {
            lse = at::empty({seqs, q_heads}, q->options().dtype(at::kFloat));
            g.lse = ptr<float>(&lse);
        }
        g.q = q->data_ptr(); g.o = o->data_ptr(); g.seq_lens = ptr<int32_t>(lens); g.q_heads = q_heads;
        g.q_stride_seq = q->stride(0); g.q_stride_head = q->stride(1); g.o_stride_seq = o->stride(0); g.o_stride_head = o->stride(1);
        g.window = window;
        g.sm_scale = x[5] == Py_None ? 1.0 / std::sqrt((double)cache.head_dim) : scale;
        int status;
        void *stream = at.stream();
        Py_BEGIN_ALLOW_THREADS
        status = attention_fn(&cache, &g, code, ENC_VARIANT_AUTO, stream);
        Py_END_ALLOW_THREADS
        if (status != ENC_OK) return PyLong_FromLong(status);
        PyObject *out = made.defined() ? THPVariable_Wrap(made) : Py_NewRef(x[7]);
        if (!return_lse || !out) return out;
        PyObject *second = THPVariable_Wrap(lse), *both = second ? PyTuple_Pack(2, out, second) : nullptr;
        Py_DECREF(out);
        Py_XDECREF(second);
        return both;
    } catch (...) {
        PyErr_Clear();
        return not_here();
    }
}

// (logits, tokens, lens, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, mask, out) -> out
PyObject *penalize_logits(PyObject *, PyObject *const *x, Py_ssize_t n) {
    if (n != 11) return not_here();
    try {
        Launch at;
        const at::Tensor *logits = at.needed(x[0]), *tokens = at.tensor(x[1]), *lens = at.tensor(x[2]), *prompts = at.tensor(x[3]);
        const at::Tensor *rep = at.tensor(x[4]), *freq = at.tensor(x[5]), *pres = at.tensor(x[6]), *ids = at.tensor(x[7]), *values = at.tensor(x[8]);
        const at::Tensor *mask = at.tensor(x[9]), *out = at.tensor(x[10]);
        if (!at.ok || logits->dim() != 2 || logits->numel() == 0 || !contiguous_rows(*logits)) return not_here();
        const int code = dtype_code(*logits);
        const int64_t m = logits->size(0), vocab = logits->size(1);
        enc_logits_args g = {};
        g.logits = logits->data_ptr(); g.rows = m; g.vocab = vocab; g.stride_in = logits->stride(0);
        if (code < 0) return not_here();
        if (tokens) {
            if (!rows(tokens, m, at::kInt) || tokens->numel() == 0 || !row(lens, m, at::kInt) || !row(prompts, m, at::kInt) || !row(rep, m, at::kFloat) ||
                !row(freq, m, at::kFloat) || !row(pres, m, at::kFloat))
                return not_here();
            g.tokens = ptr<int32_t>(tokens); g.lens = ptr<int32_t>(lens); g.prompt_lens = ptr<int32_t>(prompts);
            g.repetition = ptr<float>(rep); g.frequency = ptr<float>(freq); g.presence = ptr<float>(pres);
            g.history = tokens->size(1); g.stride_tokens = tokens->stride(0);
        } else if (lens || prompts || rep || freq || pres) {
            return not_here();
        }
        if (ids || values) {
            if (!rows(ids, m, at::kInt) || !rows(values, m, at::kFloat) || ids->sizes() != values->sizes() || ids->strides() != values->strides() ||
                ids->numel() == 0)
                return not_here();
            g.bias_ids = ptr<int32_t>(ids); g.bias_values = ptr<float>(values);
            g.num_biases = ids->size(1); g.stride_bias = ids->stride(0);
        }
        if (mask) {
            if (!rows(mask, m, at::kInt) || mask->size(1) != (vocab + 31) / 32) return not_here();
            g.mask = ptr<int32_t>(mask);
            g.stride_mask = m == 1 ? mask->size(1) : mask->stride(0);  // (a single row's stride means nothing)
        }
        at::Tensor made;
        if (out) {
            if (out->dim() != 2 || out->sizes() != logits->sizes() || !contiguous_rows(*out) || dtype_code(*out) != code || !writable(*out)) return not_here();
        } else {
            made = at::empty(logits->sizes(), logits->options());
            out = &made;
        }
        g.out = out->data_ptr();
        g.stride_out = out->stride(0);
        int status;
        void *stream = at.stream();
        Py_BEGIN_ALLOW_THREADS
        status = logits_fn(&g, code, ENC_VARIANT_AUTO, stream);
        Py_END_ALLOW_THREADS
        if (status != ENC_OK) return PyLong_FromLong(status);
        return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(x[10]);
    } catch (...) {
        PyErr_Clear();
        return not_here();
    }
}

// (addresses of enc_append_kv, enc_paged_attention, enc_paged_attention_work_bytes, enc_penalize_logits)
PyObject *init(PyObject *, PyObject *const *x, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "init() takes four addresses");
        return nullptr;
    }
    void *at[4];
    for (int i = 0; i < 4; ++i) {
        at[i] = PyLong_AsVoidPtr(x[i]);
        if (PyErr_Occurred()) return nullptr;
    }
    append_fn = reinterpret_cast<decltype(append_fn)>(at[0]);
    work_fn = reinterpret_cast<decltype(work_fn)>(at[2]);
    logits_fn = reinterpret_cast<decltype(logits_fn)>(at[3]);
    attention_fn = reinterpret_cast<decltype(attention_fn)>(at[1]);
    Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(init), FAST(append_kv), FAST(paged_attention), FAST(penalize_logits), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "enc_torch_lane", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_enc_torch_lane() { return PyModule_Create(&module); }
