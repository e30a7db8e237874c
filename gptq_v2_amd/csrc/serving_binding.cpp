// Python binding of the operators that serve a quantised decoder.  A decoder calls them once per layer and token with a few
// microseconds of work each, and there ctypes and checks written in Python take longer than the kernels do (a paged step:
// 12 us a call against 6 on the device); here the checks, the outputs and the argument struct of gptq_amd.h cost about one.
//
// No kernel and no arithmetic: tensors are checked, outputs allocated by torch, and the C entries of libgptq_amd.so called
// on the tensors' device and its current stream.  The entries' addresses come from the loader of that library (bind).
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "gptq_amd.h"

namespace {

int (*c_prompt)(const gq_attention_prompt_args *, gq_stream_t);
int (*c_append)(const gq_kv_append_args *, gq_stream_t);
size_t (*c_workspace)(int64_t, int64_t, int, int, int, int, int, int64_t);
int (*c_paged)(const gq_attention_paged_args *, gq_stream_t);
int (*c_logprobs)(const gq_token_logprobs_args *, gq_stream_t);
PyObject *check_code;   // raises what a return code of the library stands for

struct Raised {};       // a Python exception is set

template <typename... A>
[[noreturn]] void raise(PyObject *type, const char *format, A... args)
{
    PyErr_Format(type, format, args...);
    throw Raised();
}

template <typename F>
PyObject *guarded(F body)
{
    HANDLE_TH_ERRORS
    try {
        return body();
    } catch (const Raised &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

const at::Tensor &tensor(PyObject *o, const char *name)
{
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s: expected a tensor", name);
    return THPVariable_Unpack(o);
}

// an undefined tensor for None
at::Tensor optional_tensor(PyObject *o, const char *name) { return o == Py_None ? at::Tensor() : tensor(o, name); }

// Neither kind of derivative passes through these operators: tensors that carry one are refused, not cut off silently.
void no_grad(std::initializer_list<const at::Tensor *> ts)
{
    const bool back = at::GradMode::is_enabled(), forth = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    if (!back && !forth) return;
    for (const at::Tensor *t : ts) {
        if (!t->defined()) continue;
        if (back && t->requires_grad())
            raise(PyExc_RuntimeError, "this operator has no backward pass: call it under torch.no_grad() or on detached tensors");
        if (forth && t->unsafeGetTensorImpl()->autograd_meta() && t->_fw_grad(0).defined())
            raise(PyExc_RuntimeError, "this operator has no forward derivative: call it on tensors without a tangent");
    }
}

// A caller's tensor that a kernel has written: its version rises, as by any in-place operation, so that what was saved or
// kept of its old contents is known to be stale.
void written(const at::Tensor &t)
{
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int64_t half_code(const at::Tensor &t)
{
    if (t.scalar_type() == at::kHalf) return GQ_F16;
    if (t.scalar_type() == at::kBFloat16) return GQ_BF16;
    raise(PyExc_NotImplementedError, "dtype %s: only float16 and bfloat16 are supported", c10::toString(t.scalar_type()));
}

void on_gpu(const at::Tensor &t, const char *name)
{
    if (!t.is_cuda()) raise(PyExc_ValueError, "%s: must live on the GPU (got %s); there is no CPU path", name, t.device().str().c_str());
}

// A (tokens, heads, head_dim) tensor whose last dimension is dense
void rows(const at::Tensor &t, const char *name, const at::Tensor *like = nullptr)
{
    on_gpu(t, name);
    if (t.dim() != 3) raise(PyExc_ValueError, "%s: expected (tokens, heads, head_dim), got %lld dimensions", name, (long long)t.dim());
    if (t.stride(2) != 1) raise(PyExc_ValueError, "%s: the last dimension must be contiguous", name);
    if (like && (t.scalar_type() != like->scalar_type() || t.device() != like->device()))
        raise(PyExc_ValueError, "%s: is %s on %s, expected %s on %s", name, c10::toString(t.scalar_type()), t.device().str().c_str(),
              c10::toString(like->scalar_type()), like->device().str().c_str());
}

void dense(const at::Tensor &t, const char *name, at::ScalarType type, int64_t dims, const at::Tensor &like)
{
    on_gpu(t, name);
    if (!t.is_contiguous()) raise(PyExc_ValueError, "%s: must be contiguous", name);
    if (t.scalar_type() != type) raise(PyExc_ValueError, "%s: expected %s, got %s", name, c10::toString(type), c10::toString(t.scalar_type()));
    if (t.dim() != dims) raise(PyExc_ValueError, "%s: expected %lld dimensions, got %lld", name, (long long)dims, (long long)t.dim());
    if (t.device() != like.device())
        raise(PyExc_ValueError, "%s: on %s, expected %s", name, t.device().str().c_str(), like.device().str().c_str());
}

const int32_t *ints(const at::Tensor &t, const char *name, int64_t n, const at::Tensor &like)
{
    if (t.scalar_type() != at::kInt || t.device() != like.device() || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
        raise(PyExc_ValueError, "%s: expected %lld contiguous int32 on %s, got %lld %s on %s", name, (long long)n, like.device().str().c_str(),
              (long long)t.numel(), c10::toString(t.scalar_type()), t.device().str().c_str());
    return (const int32_t *)t.data_ptr();
}

const int32_t *table(const at::Tensor &t, const at::Tensor &like)
{
    if (t.dim() != 2 || t.scalar_type() != at::kInt || t.device() != like.device() || !t.is_contiguous())
        raise(PyExc_ValueError, "block_table: expected contiguous int32 (sequences, pages) on %s, got %s of %lld dimensions on %s",
              like.device().str().c_str(), c10::toString(t.scalar_type()), (long long)t.dim(), t.device().str().c_str());
    return (const int32_t *)t.data_ptr();
}

// (a dimension of size 1 has any stride)
gq_rows rows_of(const at::Tensor &t)
{
    if (!t.defined()) return {nullptr, 0, 0};
    return {t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0};
}

at::Tensor out_like(PyObject *o, const char *name, const at::Tensor &q)
{
    if (o == Py_None) return at::empty(q.sizes(), q.options());
    const at::Tensor &out = tensor(o, name);
    rows(out, name, &q);
    if (out.sizes() != q.sizes()) raise(PyExc_ValueError, "%s does not have q's shape", name);
    return out;
}

gq_paged_cache cache_of(PyObject *const *o, const at::Tensor &like)
{
    const at::Tensor &k = tensor(o[0], "cache.k"), &v = tensor(o[1], "cache.v"), &ks = tensor(o[2], "cache.k_scale"), &vs = tensor(o[3], "cache.v_scale");
    dense(k, "cache.k", at::kFloat8_e4m3fn, 4, like);
    dense(v, "cache.v", at::kFloat8_e4m3fn, 4, like);
    dense(ks, "cache.k_scale", at::kFloat, 2, like);
    dense(vs, "cache.v_scale", at::kFloat, 2, like);
    no_grad({&k, &v, &ks, &vs});
    const int64_t n = k.size(0), h = k.size(1), page = k.size(2), d = k.size(3);
    if (v.size(0) != n || v.size(1) != h || v.size(2) != d || v.size(3) != page || ks.size(0) != n || ks.size(1) != h || vs.sizes() != ks.sizes())
        raise(PyExc_ValueError, "the cache's tensors do not belong together");
    return {k.data_ptr(), v.data_ptr(), (float *)ks.data_ptr(), (float *)vs.data_ptr(), n, h, page, d};
}

double scale_of(PyObject *o, int64_t d)
{
    if (o == Py_None) return 1.0 / std::sqrt((double)d);
    const double s = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) throw Raised();
    return s;
}

int64_t integer(PyObject *o)
{
    const int64_t v = PyLong_AsLongLong(o);
    if (PyErr_Occurred()) throw Raised();
    return v;
}

bool truth(PyObject *o)
{
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised();
    return v != 0;
}

// Calls an entry on the current stream of the tensors' device; a return code becomes the exception it stands for.
template <typename A>
void call(int (*entry)(const A *, gq_stream_t), const A &args, const char *name, const at::Tensor &like)
{
    const c10::DeviceGuard guard(like.device());
    void *stream = (void *)c10::hip::getCurrentHIPStream(like.device().index()).stream();
    const int rc = entry(&args, stream);
    if (rc) {
        PyObject *r = PyObject_CallFunction(check_code, "is", rc, name);
        Py_XDECREF(r);
        if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed (code %d)", name, rc);
        throw Raised();
    }
}

void expect(Py_ssize_t got, Py_ssize_t want)
{
    if (got != want) raise(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
}

// (q, k, v, cu_seqlens, causal, scale, out)
PyObject *attention_prompt(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        expect(n, 7);
        const at::Tensor &q = tensor(o[0], "q"), &k = tensor(o[1], "k"), &v = tensor(o[2], "v");
        no_grad({&q, &k, &v});
        rows(q, "q");
        rows(k, "k", &q);
        rows(v, "v", &q);
        gq_attention_prompt_args a = {};
        a.dtype = half_code(q);
        a.n_tokens = q.size(0), a.n_heads = q.size(1), a.head_dim = q.size(2), a.n_kv_heads = k.size(1);
        if (k.sizes() != v.sizes() || k.size(0) != a.n_tokens || k.size(2) != a.head_dim || a.n_kv_heads == 0 || a.n_heads % a.n_kv_heads)
            raise(PyExc_ValueError, "q is (%lld, %lld, %lld), k (%lld, %lld, %lld), v does not fit them or the heads do not divide", (long long)a.n_tokens,
                  (long long)a.n_heads, (long long)a.head_dim, (long long)k.size(0), (long long)k.size(1), (long long)k.size(2));
        a.batch = 1;
        if (o[3] != Py_None) {
            const at::Tensor &cu = tensor(o[3], "cu_seqlens");
            a.batch = cu.numel() - 1;
            a.cu_seqlens = ints(cu, "cu_seqlens", a.batch + 1, q);
        }
        a.causal = truth(o[4]);
        a.softmax_scale = scale_of(o[5], a.head_dim);
        const at::Tensor out = out_like(o[6], "out", q);
        no_grad({&out});
        a.out = rows_of(out), a.q = rows_of(q), a.k = rows_of(k), a.v = rows_of(v);
        call(c_prompt, a, "gq_attention_prompt", q);
        written(out);
        return THPVariable_Wrap(out);
    });
}

// (cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, block_table, past_lens, cu_seqlens, q, cos, sin, interleaved, q_out)
PyObject *kv_append(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        expect(n, 14);
        const at::Tensor &k = tensor(o[4], "k"), &v = tensor(o[5], "v");
        const at::Tensor q = optional_tensor(o[9], "q"), cos = optional_tensor(o[10], "cos"), sin = optional_tensor(o[11], "sin");
        no_grad({&k, &v, &q, &cos, &sin});
        rows(k, "k");
        rows(v, "v", &k);
        gq_kv_append_args a = {};
        a.dtype = half_code(k);
        a.cache = cache_of(o, k);
        a.n_tokens = k.size(0);
        if (k.sizes() != v.sizes() || k.size(1) != a.cache.n_kv_heads || k.size(2) != a.cache.head_dim)
            raise(PyExc_ValueError, "k and v do not have the cache's %lld heads of %lld, or differ", (long long)a.cache.n_kv_heads,
                  (long long)a.cache.head_dim);
        const at::Tensor &t = tensor(o[6], "block_table");
        a.block_table = table(t, k);
        a.batch = t.size(0), a.table_width = t.size(1);
        a.past_lens = ints(tensor(o[7], "past_lens"), "past_lens", a.batch, k);
        if (o[8] != Py_None) a.cu_seqlens = ints(tensor(o[8], "cu_seqlens"), "cu_seqlens", a.batch + 1, k);
        else if (a.n_tokens != a.batch) raise(PyExc_ValueError, "%lld tokens for %lld sequences need cu_seqlens", (long long)a.n_tokens, (long long)a.batch);
        if (cos.defined() != sin.defined()) raise(PyExc_ValueError, "cos and sin belong together");
        if (cos.defined()) {
            dense(cos, "cos", at::kFloat, 2, k);
            dense(sin, "sin", at::kFloat, 2, k);
            if (cos.sizes() != sin.sizes()) raise(PyExc_ValueError, "cos and sin differ in shape");
            a.max_pos = cos.size(0), a.rotary_dim = 2 * cos.size(1);
            a.cos = (const float *)cos.data_ptr(), a.sin = (const float *)sin.data_ptr();
        }
        a.interleaved = truth(o[12]);
        at::Tensor q_out;
        if (q.defined()) {
            if (!a.rotary_dim) raise(PyExc_ValueError, "q is given to be rotated: cos and sin are missing");
            rows(q, "q", &k);
            if (q.size(0) != a.n_tokens || q.size(2) != a.cache.head_dim) raise(PyExc_ValueError, "q does not have k's tokens or head_dim");
            a.n_heads = q.size(1);
            q_out = out_like(o[13], "q_out", q);
            no_grad({&q_out});
        } else if (o[13] != Py_None) {
            raise(PyExc_ValueError, "q_out without q");
        }
        a.k = rows_of(k), a.v = rows_of(v), a.q = rows_of(q), a.q_out = rows_of(q_out);
        call(c_append, a, "gq_kv_append", k);
        for (int i = 0; i < 4; ++i) written(tensor(o[i], "cache"));
        written(q_out);
        if (!q_out.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(q_out);
    });
}

// (q, cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, seq_lens, cu_seqlens, scale, out)
PyObject *attention_paged(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        expect(n, 10);
        const at::Tensor &q = tensor(o[0], "q");
        no_grad({&q});
        rows(q, "q");
        gq_attention_paged_args a = {};
        a.dtype = half_code(q);
        a.cache = cache_of(o + 1, q);
        a.n_tokens = q.size(0), a.n_heads = q.size(1);
        if (q.size(2) != a.cache.head_dim || a.cache.n_kv_heads == 0 || a.n_heads % a.cache.n_kv_heads)
            raise(PyExc_ValueError, "q has %lld heads of %lld, the cache %lld of %lld", (long long)a.n_heads, (long long)q.size(2),
                  (long long)a.cache.n_kv_heads, (long long)a.cache.head_dim);
        const at::Tensor &t = tensor(o[5], "block_table");
        a.block_table = table(t, q);
        a.batch = t.size(0), a.table_width = t.size(1);
        a.seq_lens = ints(tensor(o[6], "seq_lens"), "seq_lens", a.batch, q);
        if (o[7] != Py_None) a.cu_seqlens = ints(tensor(o[7], "cu_seqlens"), "cu_seqlens", a.batch + 1, q);
        else if (a.n_tokens != a.batch)
            raise(PyExc_ValueError, "%lld query tokens for %lld sequences need cu_seqlens", (long long)a.n_tokens, (long long)a.batch);
        a.softmax_scale = scale_of(o[8], a.cache.head_dim);
        const at::Tensor out = out_like(o[9], "out", q);
        no_grad({&out});
        a.out = rows_of(out), a.q = rows_of(q);
        at::Tensor scratch;
        // (sizes that do not fit an int are refused by the entry itself)
        const bool fits = a.n_heads < (1 << 30) && a.cache.n_kv_heads < (1 << 30) && a.cache.head_dim < (1 << 30) && a.cache.page < (1 << 30);
        const size_t need = !fits ? 0 : c_workspace(a.n_tokens, a.batch, a.cu_seqlens != nullptr, (int)a.n_heads, (int)a.cache.n_kv_heads,
                                                    (int)a.cache.head_dim, (int)a.cache.page, a.table_width);
        if (need) {
            scratch = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
            a.workspace = scratch.data_ptr(), a.workspace_bytes = (int64_t)need;
        }
        call(c_paged, a, "gq_attention_paged", q);
        written(out);
        return THPVariable_Wrap(out);
    });
}

// (logits, tokens, top, ignore_index) -> (logprob, entropy, top_logprob or None, top_token or None)
PyObject *token_logprobs(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        expect(n, 4);
        const at::Tensor &logits = tensor(o[0], "logits");
        at::Tensor tokens = tensor(o[1], "tokens");
        no_grad({&logits});
        on_gpu(logits, "logits");
        gq_token_logprobs_args a = {};
        a.dtype = logits.scalar_type() == at::kFloat ? GQ_F32 : half_code(logits);
        const int64_t dims = logits.dim();
        if (dims == 0 || tokens.sizes() != logits.sizes().slice(0, dims - 1) || tokens.scalar_type() != at::kLong || tokens.device() != logits.device())
            raise(PyExc_ValueError, "tokens must be int64 of the logits' leading dimensions, on their device (got %s of %lld dimensions on %s)",
                  c10::toString(tokens.scalar_type()), (long long)tokens.dim(), tokens.device().str().c_str());
        a.vocab = logits.size(dims - 1), a.n_rows = tokens.numel(), a.top = integer(o[2]), a.ignore_index = integer(o[3]);
        if (a.vocab == 0 || a.top < 0 || a.top > a.vocab)
            raise(PyExc_ValueError, "%lld alternatives of %lld words", (long long)a.top, (long long)a.vocab);
        at::Tensor x = dims == 2 ? logits : logits.reshape({a.n_rows, a.vocab});
        a.row_stride = a.n_rows > 1 ? x.stride(0) : a.vocab;
        if (a.n_rows && ((a.vocab > 1 && x.stride(1) != 1) || a.row_stride < a.vocab)) {
            x = x.contiguous();
            a.row_stride = a.vocab;
        }
        if (!tokens.is_contiguous()) tokens = tokens.contiguous();
        const auto floats = logits.options().dtype(at::kFloat);
        const at::Tensor lp = at::empty(tokens.sizes(), floats), ent = at::empty(tokens.sizes(), floats);
        at::Tensor top_lp, top_tok;
        if (a.top) {
            std::vector<int64_t> shape = tokens.sizes().vec();
            shape.push_back(a.top);
            top_lp = at::empty(shape, floats);
            top_tok = at::empty(shape, tokens.options());
            a.top_logprob = (float *)top_lp.data_ptr(), a.top_token = (int64_t *)top_tok.data_ptr();
        }
        a.logits = x.data_ptr(), a.tokens = (const int64_t *)tokens.data_ptr();
        a.logprob = (float *)lp.data_ptr(), a.entropy = (float *)ent.data_ptr();
        call(c_logprobs, a, "gq_token_logprobs", logits);
        PyObject *res = PyTuple_New(4);
        if (!res) return nullptr;
        PyTuple_SET_ITEM(res, 0, THPVariable_Wrap(lp));
        PyTuple_SET_ITEM(res, 1, THPVariable_Wrap(ent));
        for (int i = 0; i < 2; ++i) {
            const at::Tensor &t = i ? top_tok : top_lp;
            if (!t.defined()) Py_INCREF(Py_None);
            PyTuple_SET_ITEM(res, 2 + i, t.defined() ? THPVariable_Wrap(t) : Py_None);
        }
        return res;
    });
}

// (addresses of gq_attention_prompt, gq_kv_append, gq_attention_paged_workspace, gq_attention_paged, gq_token_logprobs;
//  interface version of the library; what raises for a return code)
PyObject *bind(PyObject *, PyObject *const *o, Py_ssize_t n)
{
    return guarded([&]() -> PyObject * {
        expect(n, 7);
        if (integer(o[5]) != GQ_ABI_VERSION) raise(PyExc_ImportError, "the binding was built for interface version %d of the library", GQ_ABI_VERSION);
        c_prompt = (decltype(c_prompt))(uintptr_t)integer(o[0]);
        c_append = (decltype(c_append))(uintptr_t)integer(o[1]);
        c_workspace = (decltype(c_workspace))(uintptr_t)integer(o[2]);
        c_paged = (decltype(c_paged))(uintptr_t)integer(o[3]);
        c_logprobs = (decltype(c_logprobs))(uintptr_t)integer(o[4]);
        Py_INCREF(o[6]);
        Py_XSETREF(check_code, o[6]);
        Py_RETURN_NONE;
    });
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void *)bind, METH_FASTCALL, nullptr},
    {"attention_prompt", (PyCFunction)(void *)attention_prompt, METH_FASTCALL, nullptr},
    {"kv_append", (PyCFunction)(void *)kv_append, METH_FASTCALL, nullptr},
    {"attention_paged", (PyCFunction)(void *)attention_paged, METH_FASTCALL, nullptr},
    {"token_logprobs", (PyCFunction)(void *)token_logprobs, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving_binding", "Binding of the serving operators (see ops.py).", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__serving_binding() { return PyModule_Create(&module); }
