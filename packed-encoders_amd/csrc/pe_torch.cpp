// CPython extension _pe_torch: the launches of the package's kernels on torch tensors with their
// argument checks and output allocation in native code. A short batch's forward is bound by host
// time (some hundred launches of a few microseconds each); the same checks in Python cost more than
// the torch operations they replace. An attention call on 32 queries (5.7 us of kernel) takes 20.1 us
// through the torch operator and its Python body and 7.2 us from here, calls back to back; the
// 22-layer forward of 8 queries 3.84 ms with the norms and gates alone launched here, 2.99 ms with
// attention and RoPE.
//
// Each function returns None for a call it does not serve: another dtype or device, rows that are
// not 16-byte pieces, a gradient, or anything that has to see the torch operations themselves
// (autocast, tracing, function transforms, forward-mode derivatives, dispatch and function modes,
// tensor subclasses). The caller then takes the general path: torch's operations for the layer's
// norm and gate, the registered torch operators for attention and RoPE, which also raise the errors.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/autocast_mode.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <vector>

#include "../../include/pe_attn.h"
#include "../../include/pe_paged.h"

namespace {

using at::Tensor;
using c10::DispatchKey;

// Whether nothing on this thread has to see torch operations instead of a kernel launch.
bool plain_thread() {
    static const c10::DispatchKeySet watched(
        {DispatchKey::FuncTorchDynamicLayerFrontMode, DispatchKey::FuncTorchVmapMode, DispatchKey::FuncTorchGradWrapper,
         DispatchKey::FuncTorchBatched, DispatchKey::Functionalize, DispatchKey::Tracer, DispatchKey::Python,
         DispatchKey::PythonDispatcher, DispatchKey::PreDispatch});
    return !c10::impl::tls_local_dispatch_key_set().included_.has_any(watched) &&
           !at::autocast::is_autocast_enabled(at::kCUDA) && !at::impl::torch_function_mode_enabled() &&
           !c10::impl::TorchDispatchModeTLS::any_modes_set();
}

// A dense tensor on the current HIP device that records nothing and is what it says (no subclass,
// wrapper, batched stand-in without storage, lazy conjugation or forward derivative).
bool plain_any(PyObject *obj, const Tensor *&out, at::ScalarType type) {
    if (!THPVariable_CheckExact(obj)) return false;
    const Tensor &t = THPVariable_Unpack(obj);
    static const c10::DispatchKeySet wrapped({DispatchKey::FuncTorchGradWrapper, DispatchKey::FuncTorchBatched,
                                              DispatchKey::Functionalize, DispatchKey::Python, DispatchKey::Conjugate,
                                              DispatchKey::Negative, DispatchKey::ZeroTensor});
    if (!t.defined() || !t.has_storage() || !t.is_cuda() || t.scalar_type() != type || t.layout() != at::kStrided ||
        t.key_set().has_any(wrapped) || t.get_device() != c10::hip::current_device())
        return false;
    if (t.requires_grad() && c10::GradMode::is_enabled()) return false;
    if (t._fw_grad(0).defined()) return false;
    out = &t;
    return true;
}

bool aligned16(const Tensor &t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// A plain bf16 tensor, contiguous from a 16-byte boundary.
bool plain_tensor(PyObject *obj, const Tensor *&out) {
    return plain_any(obj, out, at::kBFloat16) && out->is_contiguous() && aligned16(*out);
}

// A plain bf16 [tokens, heads, head_dim] whose rows are 16-byte pieces.
bool plain_rows(PyObject *obj, const Tensor *&out) {
    return plain_any(obj, out, at::kBFloat16) && out->dim() == 3 && out->stride(2) == 1 && aligned16(*out) &&
           out->stride(0) % 8 == 0 && out->stride(1) % 8 == 0;
}

bool plain_bounds(PyObject *obj, const Tensor *&out) {
    return plain_any(obj, out, at::kInt) && out->dim() == 1 && out->is_contiguous();
}

// RoPE tables [rows, d] or [.., rows, d], both alike.
bool plain_tables(PyObject *cos_obj, PyObject *sin_obj, int64_t d, const Tensor *&cos, const Tensor *&sin) {
    return plain_tensor(cos_obj, cos) && plain_tensor(sin_obj, sin) && (cos->dim() == 2 || cos->dim() == 3) &&
           cos->size(-1) == d && cos->sizes() == sin->sizes() && cos->numel() > 0 && cos->numel() / d <= INT32_MAX;
}

hipStream_t stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// Allocations and launches run without the interpreter lock: either can wait (a full queue, an
// allocator that synchronises to free memory), and the process's other Python threads, host
// callbacks among them, go on meanwhile. Everything they need is read from the tensors before; no
// Python call is made inside.
class Unlocked {
  public:
    Unlocked() : state_(PyEval_SaveThread()) {}
    ~Unlocked() { PyEval_RestoreThread(state_); }
    Unlocked(const Unlocked &) = delete;
    Unlocked &operator=(const Unlocked &) = delete;

  private:
    PyThreadState *state_;
};

// The exception _lib.check raises for a status, or false for none.
bool failed(int status, const char *what) {
    if (status == PE_ATTN_OK) return false;
    PyErr_Format(status == PE_ATTN_ELAUNCH ? PyExc_RuntimeError : PyExc_ValueError, "%s: %s (%d)", what,
                 pe_attn_strerror(status), status);
    return true;
}

// layer_norm(x, residual or None, weight, eps) -> out, (sum, out) with a residual, or None
PyObject *layer_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "layer_norm takes x, residual, weight and eps");
        return nullptr;
    }
    const bool add = args[1] != Py_None;
    const Tensor *x = nullptr, *r = nullptr, *w = nullptr;
    if (!plain_thread() || !plain_tensor(args[0], x) || !plain_tensor(args[2], w) || (add && !plain_tensor(args[1], r)))
        Py_RETURN_NONE;
    const int64_t cols = x->dim() ? x->size(-1) : 0;
    if (cols < 8 || cols % 8 || cols > PE_LAYER_NORM_MAX_COLS || w->dim() != 1 || w->size(0) != cols ||
        (add && r->sizes() != x->sizes()))
        Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(args[3]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    const auto sizes = x->sizes().vec();
    const auto options = x->options();
    const void *src = x->const_data_ptr(), *res = add ? r->const_data_ptr() : nullptr, *weight = w->const_data_ptr();
    const int64_t rows = x->numel() / cols;
    const hipStream_t stream = stream_of(*x);
    Tensor out, sum;
    int status;
    {
        Unlocked unlocked;
        out = at::empty(sizes, options);
        if (add) sum = at::empty(sizes, options);
        status = pe_layer_norm_fwd(src, res, weight, add ? sum.mutable_data_ptr() : nullptr, out.mutable_data_ptr(), rows,
                                   (int32_t)cols, (float)eps, stream);
    }
    if (failed(status, "pe_layer_norm_fwd")) return nullptr;
    if (!add) return THPVariable_Wrap(std::move(out));
    PyObject *pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(sum)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(out)));
    return pair;
    END_HANDLE_TH_ERRORS
}

// geglu(proj) -> out, or None
PyObject *geglu(PyObject *, PyObject *arg) {
    HANDLE_TH_ERRORS
    const Tensor *x = nullptr;
    if (!plain_thread() || !plain_tensor(arg, x)) Py_RETURN_NONE;
    const int64_t both = x->dim() ? x->size(-1) : 0;
    if (both < 16 || both % 16 || both / 2 > INT32_MAX) Py_RETURN_NONE;
    auto sizes = x->sizes().vec();
    sizes.back() = both / 2;
    const auto options = x->options();
    const void *src = x->const_data_ptr();
    const int64_t rows = x->numel() / both;
    const hipStream_t stream = stream_of(*x);
    Tensor out;
    int status;
    {
        Unlocked unlocked;
        out = at::empty(sizes, options);
        status = pe_geglu_fwd(src, out.mutable_data_ptr(), rows, (int32_t)(both / 2), stream);
    }
    if (failed(status, "pe_geglu_fwd")) return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// rope_rows(positions [T] int64, max_positions, d, theta) -> (cos, sin) [1, T, d] bf16, or None
PyObject *rope_rows(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "rope_rows takes positions, max_positions, d and theta");
        return nullptr;
    }
    const int64_t max_positions = PyLong_AsLongLong(args[1]), d = PyLong_AsLongLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    const double theta = PyFloat_AsDouble(args[3]);
    if (theta == -1.0 && PyErr_Occurred()) return nullptr;
    const Tensor *pos = nullptr;
    if (max_positions < 0 || (d != 64 && d != 128 && d != 256) || !(theta > 0.0) || !plain_thread() ||
        !plain_any(args[0], pos, at::kLong) || pos->dim() != 1 || !pos->is_contiguous() || pos->numel() == 0)
        Py_RETURN_NONE;
    const int64_t sizes[3] = {1, pos->numel(), d};
    const auto options = pos->options().dtype(at::kBFloat16);
    const int64_t *positions = static_cast<const int64_t *>(pos->const_data_ptr());
    const hipStream_t stream = stream_of(*pos);
    Tensor cos, sin;
    int status;
    {
        Unlocked unlocked;
        cos = at::empty(sizes, options);
        sin = at::empty(sizes, options);
        status = pe_rope_gather_fwd(positions, max_positions, (float)theta, sizes[1], (int32_t)d, cos.mutable_data_ptr(),
                                    sin.mutable_data_ptr(), stream);
    }
    if (failed(status, "pe_rope_gather_fwd")) return nullptr;
    PyObject *pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(cos)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(sin)));
    return pair;
    END_HANDLE_TH_ERRORS
}

// rope(qkv [.., 3 h d], h, d, cos, sin) -> (q, k) [.., h, d], or None
PyObject *rope(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "rope takes qkv, h, d, cos and sin");
        return nullptr;
    }
    const int64_t h = PyLong_AsLongLong(args[1]), d = PyLong_AsLongLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    const Tensor *qkv = nullptr, *cos = nullptr, *sin = nullptr;
    if (h < 1 || h > (1 << 20) || (d != 64 && d != 128 && d != 256) || !plain_thread() || !plain_tensor(args[0], qkv) ||
        !plain_tables(args[3], args[4], d, cos, sin))
        Py_RETURN_NONE;
    const int64_t width = 3 * h * d;
    if (!qkv->dim() || qkv->size(-1) != width || qkv->numel() == 0 || qkv->numel() / width > INT32_MAX) Py_RETURN_NONE;
    auto sizes = qkv->sizes().vec();
    sizes.back() = h;
    sizes.push_back(d);
    const auto options = qkv->options();
    const hipStream_t stream = stream_of(*qkv);
    pe_rope_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.dtype = PE_ATTN_DTYPE_BF16;
    a.qkv = qkv->const_data_ptr();
    a.cos = cos->const_data_ptr();
    a.sin = sin->const_data_ptr();
    a.qkv_stride_row = width;
    a.table_stride_row = d;
    a.table_rows = (int32_t)(cos->numel() / d);
    a.n_rows = (int32_t)(qkv->numel() / width);
    a.n_heads = (int32_t)h;
    a.head_dim = (int32_t)d;
    Tensor q, k;
    int status;
    {
        Unlocked unlocked;
        q = at::empty(sizes, options);
        k = at::empty(sizes, options);
        a.q_out = q.mutable_data_ptr();
        a.k_out = k.mutable_data_ptr();
        status = pe_rope_qkv_fwd(&a, stream);
    }
    if (failed(status, "pe_rope_qkv_fwd")) return nullptr;
    PyObject *pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(q)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(k)));
    return pair;
    END_HANDLE_TH_ERRORS
}

// The attention calls' arguments past their tensors, in the order Python passes them.
struct Options {
    int64_t max_seqlen, window_left, window_right, causal, short_max, max_seqlen_k, band_kernel, min_seqlen;
    double scale;
    void *args;  // a pe_attn_args to fill instead of launching, or NULL

    // false with a Python exception set, or (ok = false) for a value no kernel argument holds
    bool parse(PyObject *const *a, bool &ok) {
        int64_t *ints[8] = {&max_seqlen, &window_left, &window_right, &causal, &short_max, &max_seqlen_k, &band_kernel,
                            &min_seqlen};
        ok = true;
        for (int i = 0; i < 8; ++i) {
            *ints[i] = PyLong_AsLongLong(a[i]);
            if (*ints[i] == -1 && PyErr_Occurred()) return false;
            ok = ok && *ints[i] >= INT32_MIN && *ints[i] <= INT32_MAX;
        }
        scale = PyFloat_AsDouble(a[8]);
        if (scale == -1.0 && PyErr_Occurred()) return false;
        args = PyLong_AsVoidPtr(a[9]);
        return args || !PyErr_Occurred();
    }
    static constexpr int kCount = 10;
};

// Completes `a` (q, k, v and the tables filled in), allocates the output shaped `sizes` and either
// launches the whole call, returning the output, or hands the arguments over: (output, stream).
PyObject *finish(pe_attn_args &a, const Options &o, const Tensor &like, at::IntArrayRef sizes, const Tensor &cu) {
    a.struct_size = sizeof(a);
    a.dtype = PE_ATTN_DTYPE_BF16;
    a.cu_seqlens = static_cast<const int32_t *>(cu.const_data_ptr());
    a.n_seq = (int32_t)(cu.numel() - 1);
    a.max_seqlen = (int32_t)o.max_seqlen;
    a.softmax_scale = (float)o.scale;
    a.window_left = (int32_t)o.window_left;
    a.window_right = (int32_t)o.window_right;
    a.causal = o.causal ? 1 : 0;
    a.short_max = (int32_t)o.short_max;
    a.band_kernel = (int32_t)o.band_kernel;
    a.min_seqlen = (int32_t)o.min_seqlen;
    a.o_stride_head = a.head_dim;
    a.o_stride_token = (int64_t)a.n_heads_q * a.head_dim;
    const auto shape = sizes.vec();
    const auto options = like.options();
    const hipStream_t stream = stream_of(like);
    Tensor out, workspace;
    const char *what = "pe_attn_workspace_size";
    int status = PE_ATTN_OK;
    {
        Unlocked unlocked;
        out = at::empty(shape, options);
        a.o = out.mutable_data_ptr();
        size_t bytes = 0;
        if (!o.args) status = pe_attn_workspace_size(&a, &bytes);
        if (!o.args && status == PE_ATTN_OK) {
            if (bytes) workspace = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
            what = "pe_varlen_attn_fwd";
            status = pe_varlen_attn_fwd(&a, bytes ? workspace.mutable_data_ptr() : nullptr, bytes, stream);
        }
    }
    if (failed(status, what)) return nullptr;
    if (o.args) {
        std::memcpy(o.args, &a, sizeof(a));
        PyObject *pair = PyTuple_New(2);
        if (!pair) return nullptr;
        PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(out)));
        PyTuple_SET_ITEM(pair, 1, PyLong_FromVoidPtr(stream));
        return pair;
    }
    return THPVariable_Wrap(std::move(out));
}

// attention(q, k, v, cu, gate or None, cu_k or None, cos or None, sin or None, *Options)
PyObject *attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8 + Options::kCount) {
        PyErr_SetString(PyExc_TypeError, "attention takes its eight tensors and ten options");
        return nullptr;
    }
    Options o;
    bool ok;
    if (!o.parse(args + 8, ok)) return nullptr;
    const Tensor *q = nullptr, *k = nullptr, *v = nullptr, *cu = nullptr, *g = nullptr, *cuk = nullptr, *cos = nullptr,
                 *sin = nullptr;
    const bool gated = args[4] != Py_None, own_keys = args[5] != Py_None, rotate = args[6] != Py_None;
    if (!ok || !plain_thread() || !plain_rows(args[0], q) || !plain_rows(args[1], k) || !plain_rows(args[2], v) ||
        !plain_bounds(args[3], cu) || (gated && !plain_rows(args[4], g)) || (own_keys && !plain_bounds(args[5], cuk)) ||
        rotate != (args[7] != Py_None) || (rotate && !plain_tables(args[6], args[7], q->size(2), cos, sin)))
        Py_RETURN_NONE;
    const int64_t hkv = k->size(1);
    if (k->sizes() != v->sizes() || q->size(2) != k->size(2) || (!own_keys && q->size(0) != k->size(0)) || hkv < 1 ||
        q->size(1) % hkv || (gated && g->sizes() != q->sizes()) || (own_keys && cuk->numel() != cu->numel()) ||
        q->size(0) == 0 || q->size(0) > INT32_MAX || k->size(0) > INT32_MAX || q->size(1) > INT32_MAX ||
        q->size(2) > 256 || cu->numel() < 2 || cu->numel() > INT32_MAX)
        Py_RETURN_NONE;
    pe_attn_args a;
    std::memset(&a, 0, sizeof(a));
    a.q = q->const_data_ptr();
    a.k = k->const_data_ptr();
    a.v = v->const_data_ptr();
    a.q_stride_token = q->stride(0);
    a.q_stride_head = q->stride(1);
    a.k_stride_token = k->stride(0);
    a.k_stride_head = k->stride(1);
    a.v_stride_token = v->stride(0);
    a.v_stride_head = v->stride(1);
    if (gated) {
        a.gate = g->const_data_ptr();
        a.gate_stride_token = g->stride(0);
        a.gate_stride_head = g->stride(1);
    }
    a.total_tokens = (int32_t)q->size(0);
    a.n_heads_q = (int32_t)q->size(1);
    a.n_heads_kv = (int32_t)hkv;
    a.head_dim = (int32_t)q->size(2);
    if (own_keys) {
        a.cu_seqlens_k = static_cast<const int32_t *>(cuk->const_data_ptr());
        a.total_tokens_k = (int32_t)k->size(0);
        a.max_seqlen_k = (int32_t)o.max_seqlen_k;
    }
    if (rotate) {
        a.rope_cos = cos->const_data_ptr();
        a.rope_sin = sin->const_data_ptr();
        a.rope_table_stride = a.head_dim;
        a.rope_table_rows = (int32_t)(cos->numel() / a.head_dim);
    }
    return finish(a, o, *q, q->sizes(), *cu);
    END_HANDLE_TH_ERRORS
}

// attention_qkv(qkv [1, tokens, 3 h d], h, d, cu, cos, sin, *Options): RoPE and attention from the
// packed projection, the output [1, tokens, h d]
PyObject *attention_qkv(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 + Options::kCount) {
        PyErr_SetString(PyExc_TypeError, "attention_qkv takes qkv, h, d, cu, cos, sin and ten options");
        return nullptr;
    }
    Options o;
    bool ok;
    if (!o.parse(args + 6, ok)) return nullptr;
    const int64_t h = PyLong_AsLongLong(args[1]), d = PyLong_AsLongLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    const Tensor *qkv = nullptr, *cu = nullptr, *cos = nullptr, *sin = nullptr;
    if (!ok || h < 1 || h > (1 << 20) || (d != 64 && d != 128) || !plain_thread() || !plain_tensor(args[0], qkv) ||
        !plain_bounds(args[3], cu) || !plain_tables(args[4], args[5], d, cos, sin))
        Py_RETURN_NONE;
    const int64_t width = 3 * h * d;
    if (qkv->dim() != 3 || qkv->size(0) != 1 || qkv->size(2) != width || qkv->size(1) == 0 || qkv->size(1) > INT32_MAX ||
        cu->numel() < 2 || cu->numel() > INT32_MAX)
        Py_RETURN_NONE;
    pe_attn_args a;
    std::memset(&a, 0, sizeof(a));
    const char *base = static_cast<const char *>(qkv->const_data_ptr());
    a.q = base;
    a.k = base + 2 * h * d;
    a.v = base + 4 * h * d;
    a.q_stride_token = a.k_stride_token = a.v_stride_token = width;
    a.q_stride_head = a.k_stride_head = a.v_stride_head = d;
    a.total_tokens = (int32_t)qkv->size(1);
    a.n_heads_q = a.n_heads_kv = (int32_t)h;
    a.head_dim = (int32_t)d;
    a.rope_cos = cos->const_data_ptr();
    a.rope_sin = sin->const_data_ptr();
    a.rope_table_stride = d;
    a.rope_table_rows = (int32_t)(cos->numel() / d);
    const int64_t sizes[3] = {1, qkv->size(1), h * d};
    return finish(a, o, *qkv, sizes, *cu);
    END_HANDLE_TH_ERRORS
}

// rotary(x, positions, inv_freq, interleaved, inverse, scale) -> out, or None. x [tokens, heads, d] with any
// strides that leave d whole, or contiguous of more axes; positions one per token.
PyObject *rotary(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) {
        PyErr_SetString(PyExc_TypeError, "rotary takes x, positions, inv_freq, interleaved, inverse and scale");
        return nullptr;
    }
    const double scale = PyFloat_AsDouble(args[5]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    const Tensor *x = nullptr, *pos = nullptr, *freq = nullptr;
    if (!plain_thread() || !THPVariable_CheckExact(args[0]) || !THPVariable_CheckExact(args[1])) Py_RETURN_NONE;
    const at::ScalarType type = THPVariable_Unpack(args[0]).scalar_type();
    const at::ScalarType index = THPVariable_Unpack(args[1]).scalar_type();
    const int32_t dtype = type == at::kBFloat16 ? PE_ROTARY_BF16
                          : type == at::kHalf   ? PE_ROTARY_FP16
                          : type == at::kFloat  ? PE_ROTARY_FP32
                                                : 0;
    if (!dtype || (index != at::kLong && index != at::kInt) || !plain_any(args[0], x, type) ||
        !plain_any(args[1], pos, index) || !plain_any(args[2], freq, at::kFloat) || x->dim() < 3 || x->numel() == 0 ||
        freq->dim() != 1 || !freq->is_contiguous() || !pos->is_contiguous())
        Py_RETURN_NONE;
    const int64_t dims = x->dim(), d = x->size(dims - 1), heads = x->size(dims - 2), half = freq->numel();
    const bool rows = dims == 3 && x->stride(2) == 1;
    if ((!rows && !x->is_contiguous()) || pos->dim() != dims - 2 || pos->sizes() != x->sizes().slice(0, dims - 2) ||
        half < 1 || half > PE_ROTARY_MAX_PAIRS || 2 * half > d || d > INT32_MAX || heads > INT32_MAX)
        Py_RETURN_NONE;
    const auto sizes = x->sizes().vec();
    const auto options = x->options();
    const hipStream_t stream = stream_of(*x);
    pe_rotary_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.dtype = dtype;
    a.x = x->const_data_ptr();
    a.positions = pos->const_data_ptr();
    a.inv_freq = static_cast<const float *>(freq->const_data_ptr());
    a.x_stride_token = rows ? x->stride(0) : heads * d;
    a.x_stride_head = rows ? x->stride(1) : d;
    a.n_tokens = x->numel() / (heads * d);
    a.n_heads = (int32_t)heads;
    a.head_dim = (int32_t)d;
    a.half = (int32_t)half;
    a.positions_32 = index == at::kInt;
    a.interleaved = args[3] == Py_True;
    a.inverse = args[4] == Py_True;
    a.scale = (float)scale;
    Tensor out;
    int status;
    {
        Unlocked unlocked;
        out = at::empty(sizes, options);
        a.out = out.mutable_data_ptr();
        status = pe_rotary_fwd(&a, stream);
    }
    if (failed(status, "pe_rotary_fwd")) return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// The pages and what finds them: [n_pages, page_size, heads, d] bf16 twice, int32 table, cu_seqlens, seqlens_k.
struct Pages {
    const Tensor *k = nullptr, *v = nullptr, *table = nullptr, *cu = nullptr, *lens = nullptr;

    static bool rows(PyObject *obj, const Tensor *&out) {
        return plain_any(obj, out, at::kBFloat16) && out->dim() == 4 && out->stride(3) == 1 && aligned16(*out) &&
               out->stride(0) % 8 == 0 && out->stride(1) % 8 == 0 && out->stride(2) % 8 == 0;
    }
    bool parse(PyObject *const *a) {
        if (!rows(a[0], k) || !rows(a[1], v) || k->sizes() != v->sizes() || !plain_any(a[2], table, at::kInt) ||
            table->dim() != 2 || !plain_bounds(a[3], cu) || !plain_bounds(a[4], lens))
            return false;
        const int64_t n = cu->numel() - 1;
        if (n < 1 || n > INT32_MAX || lens->numel() != n || table->size(0) != n || table->size(1) > INT32_MAX ||
            (table->size(1) > 1 && table->stride(1) != 1))
            return false;
        for (int i = 0; i < 4; ++i)
            if (k->size(i) > INT32_MAX) return false;
        return k->size(1) >= PE_PAGED_PAGE_MULTIPLE && k->size(1) % PE_PAGED_PAGE_MULTIPLE == 0 && k->size(2) >= 1;
    }
};

// paged_attention(q, k_pages, v_pages, table, cu, lens, max_seqlen, max_seqlen_k, scale, window_left, window_right,
// causal) -> out, or None
PyObject *paged_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 12) {
        PyErr_SetString(PyExc_TypeError, "paged_attention takes its six tensors and six options");
        return nullptr;
    }
    const int at_int[4] = {6, 7, 9, 10};
    int64_t ints[4];
    bool fits = true;
    for (int i = 0; i < 4; ++i) {
        ints[i] = PyLong_AsLongLong(args[at_int[i]]);
        if (ints[i] == -1 && PyErr_Occurred()) return nullptr;
        fits = fits && ints[i] >= INT32_MIN && ints[i] <= INT32_MAX;
    }
    const double scale = PyFloat_AsDouble(args[8]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    const Tensor *q = nullptr;
    Pages pages;
    if (!fits || !plain_thread() || !plain_rows(args[0], q) || !pages.parse(args + 1)) Py_RETURN_NONE;
    const Tensor &k = *pages.k, &v = *pages.v;
    if (q->size(2) != k.size(3) || q->size(1) < 1 || q->size(1) % k.size(2) || q->size(0) == 0 || q->size(0) > INT32_MAX ||
        q->size(1) > INT32_MAX)
        Py_RETURN_NONE;
    pe_paged_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.dtype = PE_ATTN_DTYPE_BF16;
    a.q = q->const_data_ptr();
    a.k_pages = k.const_data_ptr();
    a.v_pages = v.const_data_ptr();
    a.page_table = static_cast<const int32_t *>(pages.table->const_data_ptr());
    a.cu_seqlens = static_cast<const int32_t *>(pages.cu->const_data_ptr());
    a.seqlens_k = static_cast<const int32_t *>(pages.lens->const_data_ptr());
    a.q_stride_token = q->stride(0);
    a.q_stride_head = q->stride(1);
    a.k_stride_page = k.stride(0);
    a.k_stride_token = k.stride(1);
    a.k_stride_head = k.stride(2);
    a.v_stride_page = v.stride(0);
    a.v_stride_token = v.stride(1);
    a.v_stride_head = v.stride(2);
    a.o_stride_head = q->size(2);
    a.o_stride_token = q->size(1) * q->size(2);
    a.table_stride = pages.table->stride(0);
    a.n_seq = (int32_t)pages.lens->numel();
    a.total_tokens = (int32_t)q->size(0);
    a.max_seqlen = (int32_t)ints[0];
    a.max_seqlen_k = (int32_t)ints[1];
    a.n_heads_q = (int32_t)q->size(1);
    a.n_heads_kv = (int32_t)k.size(2);
    a.head_dim = (int32_t)q->size(2);
    a.n_pages = (int32_t)k.size(0);
    a.page_size = (int32_t)k.size(1);
    a.max_pages = (int32_t)pages.table->size(1);
    a.softmax_scale = (float)scale;
    a.window_left = (int32_t)ints[2];
    a.window_right = (int32_t)ints[3];
    a.causal = args[11] == Py_True;
    const auto sizes = q->sizes().vec();
    const auto options = q->options();
    const hipStream_t stream = stream_of(*q);
    Tensor out, workspace;
    const char *what = "pe_paged_workspace_size";
    int status;
    {
        Unlocked unlocked;
        out = at::empty(sizes, options);
        a.o = out.mutable_data_ptr();
        size_t bytes = 0;
        status = pe_paged_workspace_size(&a, &bytes);
        if (status == PE_ATTN_OK) {
            if (bytes) workspace = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
            what = "pe_paged_attn_fwd";
            status = pe_paged_attn_fwd(&a, bytes ? workspace.mutable_data_ptr() : nullptr, bytes, stream);
        }
    }
    if (failed(status, what)) return nullptr;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// paged_append(q or None, k, v, k_pages, v_pages, table, cu, lens, inv_freq or None, interleaved, rope_scale) -> the
// rotated q (True without q), or None
PyObject *paged_append(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11) {
        PyErr_SetString(PyExc_TypeError, "paged_append takes nine tensors, interleaved and rope_scale");
        return nullptr;
    }
    const double scale = PyFloat_AsDouble(args[10]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    const bool queries = args[0] != Py_None, turns = args[8] != Py_None;
    const Tensor *q = nullptr, *k = nullptr, *v = nullptr, *freq = nullptr;
    Pages pages;
    if (!plain_thread() || (queries && !plain_rows(args[0], q)) || !plain_rows(args[1], k) || !plain_rows(args[2], v) ||
        !pages.parse(args + 3) || (turns && !plain_any(args[8], freq, at::kFloat)))
        Py_RETURN_NONE;
    const int64_t d = k->size(2), half = turns ? freq->numel() : 0;
    if (k->sizes() != v->sizes() || k->size(1) != pages.k->size(2) || d != pages.k->size(3) || d % 8 || k->size(0) == 0 ||
        k->size(0) > INT32_MAX ||
        (queries && (q->size(0) != k->size(0) || q->size(2) != d || q->size(1) < 1 || q->size(1) > INT32_MAX)) ||
        (turns && (freq->dim() != 1 || !freq->is_contiguous() || half < 1 || half > PE_ROTARY_MAX_PAIRS || 2 * half > d)))
        Py_RETURN_NONE;
    pe_append_args a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.dtype = PE_ATTN_DTYPE_BF16;
    a.k = k->const_data_ptr();
    a.v = v->const_data_ptr();
    a.page_table = static_cast<const int32_t *>(pages.table->const_data_ptr());
    a.cu_seqlens = static_cast<const int32_t *>(pages.cu->const_data_ptr());
    a.seqlens_k = static_cast<const int32_t *>(pages.lens->const_data_ptr());
    a.inv_freq = turns ? static_cast<const float *>(freq->const_data_ptr()) : nullptr;
    a.k_stride_token = k->stride(0);
    a.k_stride_head = k->stride(1);
    a.v_stride_token = v->stride(0);
    a.v_stride_head = v->stride(1);
    a.kp_stride_page = pages.k->stride(0);
    a.kp_stride_token = pages.k->stride(1);
    a.kp_stride_head = pages.k->stride(2);
    a.vp_stride_page = pages.v->stride(0);
    a.vp_stride_token = pages.v->stride(1);
    a.vp_stride_head = pages.v->stride(2);
    a.table_stride = pages.table->stride(0);
    a.n_seq = (int32_t)pages.lens->numel();
    a.total_tokens = (int32_t)k->size(0);
    a.n_heads_kv = (int32_t)k->size(1);
    a.head_dim = (int32_t)d;
    a.n_pages = (int32_t)pages.k->size(0);
    a.page_size = (int32_t)pages.k->size(1);
    a.max_pages = (int32_t)pages.table->size(1);
    a.half = (int32_t)half;
    a.interleaved = args[9] == Py_True;
    a.rope_scale = (float)scale;
    a.k_pages = pages.k->mutable_data_ptr();
    a.v_pages = pages.v->mutable_data_ptr();
    const auto options = k->options();
    const hipStream_t stream = stream_of(*k);
    int64_t sizes[3] = {0, 0, 0};
    if (queries) {
        a.q = q->const_data_ptr();
        a.q_stride_token = q->stride(0);
        a.q_stride_head = q->stride(1);
        a.n_heads_q = (int32_t)q->size(1);
        for (int i = 0; i < 3; ++i) sizes[i] = q->size(i);
    }
    Tensor out;
    int status;
    {
        Unlocked unlocked;
        if (queries) {
            out = at::empty(at::IntArrayRef(sizes, 3), options);
            a.q_out = out.mutable_data_ptr();
        }
        status = pe_paged_append_fwd(&a, stream);
    }
    if (failed(status, "pe_paged_append_fwd")) return nullptr;
    if (!queries) Py_RETURN_TRUE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// Python integers of a list into `out`; false, with no exception left, for anything else.
bool page_list(PyObject *list, std::vector<int32_t> &out) {
    if (!PyList_CheckExact(list)) return false;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    out.resize(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const int64_t x = PyLong_AsLongLong(PyList_GET_ITEM(list, i));
        if (x == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            return false;
        }
        if (x < 0 || x > INT32_MAX) return false;
        out[i] = (int32_t)x;
    }
    return true;
}

// copy_pages([caches], [src], [dst]) -> True, or None. Contiguous caches of one shape and type.
PyObject *copy_pages(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3 || !PyList_CheckExact(args[0])) {
        PyErr_SetString(PyExc_TypeError, "copy_pages takes lists of caches, sources and targets");
        return nullptr;
    }
    const Py_ssize_t count = PyList_GET_SIZE(args[0]);
    std::vector<int32_t> src, dst;
    if (!plain_thread() || count < 1 || !page_list(args[1], src) || !page_list(args[2], dst) || src.size() != dst.size() ||
        src.size() > INT32_MAX)
        Py_RETURN_NONE;
    std::vector<void *> bases;
    int64_t pages = 0, page_bytes = 0;
    hipStream_t stream = nullptr;
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject *obj = PyList_GET_ITEM(args[0], i);
        const Tensor *t = nullptr;
        if (!THPVariable_CheckExact(obj) || !plain_any(obj, t, THPVariable_Unpack(obj).scalar_type()) || t->dim() < 4 ||
            !t->is_contiguous() || t->numel() == 0)
            Py_RETURN_NONE;
        const int64_t dims = t->dim(), at = t->size(dims - 4);
        const int64_t bytes = t->size(dims - 3) * t->size(dims - 2) * t->size(dims - 1) * (int64_t)t->element_size();
        if (i && (at != pages || bytes != page_bytes)) Py_RETURN_NONE;
        pages = at;
        page_bytes = bytes;
        const int64_t caches = (int64_t)t->nbytes() / (at * bytes);
        if (pages > INT32_MAX || (int64_t)bases.size() + caches > INT32_MAX) Py_RETURN_NONE;
        char *base = static_cast<char *>(t->mutable_data_ptr());
        for (int64_t c = 0; c < caches; ++c) bases.push_back(base + c * at * bytes);
        stream = stream_of(*t);
    }
    int status;
    {
        Unlocked unlocked;
        status = pe_copy_pages(bases.data(), (int32_t)bases.size(), page_bytes, page_bytes, (int32_t)pages, src.data(),
                               dst.data(), (int32_t)src.size(), stream);
    }
    if (failed(status, "pe_copy_pages")) return nullptr;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

#define PE_FASTCALL(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL

PyMethodDef methods[] = {
    {"layer_norm", PE_FASTCALL(layer_norm), "layer_norm(x, residual, weight, eps) -> out, (sum, out) or None"},
    {"geglu", geglu, METH_O, "geglu(proj) -> out or None"},
    {"rope_rows", PE_FASTCALL(rope_rows), "rope_rows(positions, max_positions, d, theta) -> (cos, sin) or None"},
    {"rope", PE_FASTCALL(rope), "rope(qkv, h, d, cos, sin) -> (q, k) or None"},
    {"attention", PE_FASTCALL(attention),
     "attention(q, k, v, cu, gate, cu_k, cos, sin, max_seqlen, window_left, window_right, causal, short_max, "
     "max_seqlen_k, band_kernel, min_seqlen, scale, args) -> out, (out, stream) or None"},
    {"attention_qkv", PE_FASTCALL(attention_qkv),
     "attention_qkv(qkv, h, d, cu, cos, sin, max_seqlen, window_left, window_right, causal, short_max, max_seqlen_k, "
     "band_kernel, min_seqlen, scale, args) -> out, (out, stream) or None"},
    {"rotary", PE_FASTCALL(rotary), "rotary(x, positions, inv_freq, interleaved, inverse, scale) -> out or None"},
    {"paged_attention", PE_FASTCALL(paged_attention),
     "paged_attention(q, k_pages, v_pages, table, cu, lens, max_seqlen, max_seqlen_k, scale, window_left, window_right, "
     "causal) -> out or None"},
    {"paged_append", PE_FASTCALL(paged_append),
     "paged_append(q, k, v, k_pages, v_pages, table, cu, lens, inv_freq, interleaved, rope_scale) -> q, True or None"},
    {"copy_pages", PE_FASTCALL(copy_pages), "copy_pages(caches, src, dst) -> True or None"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pe_torch", "Native launches of the package's kernels on torch tensors", -1,
                      methods};

}  // namespace

PyMODINIT_FUNC PyInit__pe_torch() {
    if (pe_attn_abi_version() != PE_ATTN_ABI_VERSION) {
        PyErr_Format(PyExc_ImportError, "_pe_torch was built for ABI %d of libpe_attn.so, which has %d", PE_ATTN_ABI_VERSION,
                     pe_attn_abi_version());
        return nullptr;
    }
    return PyModule_Create(&module);
}
