// The per-call host path of the two operators that every projection goes through, and of those on 8-bit caches, 8-bit weights and logits, as a CPython
// extension over the C ABI: argument checks, allocation of results and workspace, the choice of the kernel family, the launches.
//
// What bounds a small call is this path and not the GPU: written in Python over ctypes, a projection of one token took 20 us
// of host time (device guard 1.5, stream look-up 3.2, three allocations, twenty converted arguments) around a kernel of
// five; here it takes about seven, of which the launch itself is three.  (Written in Python the operators on 8-bit caches, weights and logits took 16 to 20 us a call around kernels of 2 to 10.)
#include <torch/csrc/python_headers.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "../../include/wf_b200.h"

namespace {

struct PyFailure {};  // a Python exception is set

[[noreturn]] void raise(PyObject* type, const std::string& msg) {
    PyErr_SetString(type, msg.c_str());
    throw PyFailure();
}

// Messages without a stream: where the compiler links its own libstdc++ into this library, a number put into a stream of it meets the facets of torch's,
// and the process ends instead of the exception being raised.
std::string text(const char* v) { return v; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(int v) { return std::to_string(v); }
std::string text(at::ScalarType v) { return c10::toString(v); }
std::string text(at::IntArrayRef v) {
    std::string s = "[";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + "]";
}
template <class... Parts>
std::string message(const Parts&... parts) {
    std::string s;
    ((s += text(parts)), ...);
    return s;
}

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return WF_F32;
        case at::kHalf: return WF_F16;
        case at::kBFloat16: return WF_BF16;
        case at::kChar: return WF_I8;
        default: raise(PyExc_KeyError, message("unsupported dtype ", t));
    }
}

const at::Tensor* optional_tensor(PyObject* o) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "expected a tensor or None");
    return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o) {
    const at::Tensor* t = optional_tensor(o);
    if (!t) raise(PyExc_TypeError, "expected a tensor, got None");
    return *t;
}
void need_cuda(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        if (t && !t->is_cuda()) raise(PyExc_RuntimeError, "wf_b200 operators need CUDA tensors (there is no CPU path)");
}
long long_arg(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw PyFailure();
    return v;
}
double float_arg(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PyFailure();
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PyFailure();
    return v != 0;
}
void check(int rc, const char* what) {
    if (rc) raise(PyExc_RuntimeError, message(what, " failed (code ", rc, "): ", wf_last_error()));
}

// x as [tokens, K] with unit inner stride
at::Tensor as_rows(const at::Tensor& x) {
    if (x.dim() == 0) raise(PyExc_IndexError, "expected a tensor with at least one dimension");
    at::Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    return r.stride(1) == 1 ? r : r.contiguous();
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Quantized {
    at::Tensor q, scale, rowsum;
};
Quantized quantize(const at::Tensor& rows, bool per_tensor, double eps, bool want_rowsum, void* stream) {
    const int64_t m = rows.size(0), k = rows.size(1);
    Quantized r;
    r.q = at::empty({m, k}, rows.options().dtype(at::kChar));
    r.scale = at::empty({per_tensor ? 1 : m}, rows.options().dtype(at::kFloat));
    if (want_rowsum) r.rowsum = at::empty({m}, rows.options().dtype(at::kInt));
    const int dt = dtype_code(rows.scalar_type());
    const int64_t ldx = rows.stride(0);
    int rc;
    {
        pybind11::gil_scoped_release nogil;
        rc = wf_act_quant_i8(rows.data_ptr(), dt, m, k, ldx, per_tensor ? WF_ACT_PER_TENSOR : WF_ACT_PER_TOKEN, static_cast<float>(eps),
                             static_cast<int8_t*>(r.q.data_ptr()), static_cast<float*>(r.scale.data_ptr()), static_cast<int32_t*>(ptr(r.rowsum)), stream);
    }
    check(rc, "wf_act_quant_i8");
    return r;
}

// The contraction's workspace, one of the call's own: two streams of a device never write the same tokens.  The form for many
// tokens wants room for one byte per weight; on a card that has none left the call runs the packed form in the smaller one.
at::Tensor contraction_workspace(int64_t m, int64_t n, int64_t k, const at::TensorOptions& bytes) {
    const int64_t most = static_cast<int64_t>(wf_prefill_workspace_bytes_for(m, n, k)), least = static_cast<int64_t>(wf_prefill_workspace_bytes(m, k));
    if (most > least) {
        try {
            return at::empty({most}, bytes);
        } catch (const c10::OutOfMemoryError&) {
        }
    }
    return at::empty({least}, bytes);
}

PyObject* wrap(const at::Tensor& t) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) throw PyFailure();
    return o;
}
PyObject* wrap_all(std::initializer_list<at::Tensor> ts) {
    PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
    if (!out) throw PyFailure();
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) {
        PyObject* o = THPVariable_Wrap(t);
        if (!o) {
            Py_DECREF(out);
            throw PyFailure();
        }
        PyTuple_SET_ITEM(out, i++, o);
    }
    return out;
}

// act_quant_i8(x, per_tensor, eps, want_rowsum) -> (q, scale[, rowsum])
PyObject* act_quant_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        if (n != 4) raise(PyExc_TypeError, "act_quant_i8 takes 4 arguments");
        const at::Tensor& x = tensor(a[0]);
        need_cuda({&x});
        const at::Tensor rows = as_rows(x);
        c10::cuda::CUDAGuard guard(x.device());
        const Quantized r = quantize(rows, truth(a[1]), float_arg(a[2]), truth(a[3]), c10::cuda::getCurrentCUDAStream().stream());
        const at::Tensor q = x.dim() == 2 ? r.q : r.q.reshape(x.sizes());
        return r.rowsum.defined() ? wrap_all({q, r.scale, r.rowsum}) : wrap_all({q, r.scale});
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// bitlinear(x, codes, w_scale, bias, out_dtype, layout, x_scale, eps, want_acc, flags, path, out, decode_max_tokens,
//           prequant_min_tokens, prequant_min_elems) -> y | (y, acc);   path: 0 auto, 1 decode, 2 prefill
PyObject* bitlinear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    try {
        if (n_args != 15) raise(PyExc_TypeError, "bitlinear takes 15 arguments");
        const at::Tensor& x = tensor(a[0]);
        at::Tensor codes = tensor(a[1]);
        const at::Tensor* bias = optional_tensor(a[3]);
        const at::Tensor* x_scale = optional_tensor(a[6]);
        const at::Tensor* out = optional_tensor(a[11]);
        need_cuda({&x, &codes, bias, x_scale});
        if (x.dim() == 0) raise(PyExc_IndexError, "bitlinear: x needs at least one dimension");
        const int64_t k = x.size(-1);
        if (codes.scalar_type() != at::kByte || codes.dim() != 2 || codes.size(1) * 4 != k)
            raise(PyExc_ValueError, message("codes must be uint8 [N, K/4] with K=", k, ", got ", codes.sizes(), " ", codes.scalar_type()));
        const int64_t n = codes.size(0);
        at::Tensor rows = as_rows(x);
        const int64_t m = rows.size(0);
        c10::cuda::CUDAGuard guard(x.device());
        at::ScalarType y_type = x.scalar_type() == at::kChar ? at::kFloat : x.scalar_type();
        if (a[4] != Py_None) {
            if (!THPDtype_Check(a[4])) raise(PyExc_TypeError, "out_dtype must be a torch.dtype");
            y_type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
        }
        const at::Tensor y = out ? *out : at::empty({m, n}, x.options().dtype(y_type));
        at::Tensor acc;
        if (truth(a[8])) acc = at::empty({m, n}, x.options().dtype(at::kInt));
        const float* ws_dev = nullptr;
        float ws_host = 0.f;
        if (THPVariable_Check(a[2])) {
            const at::Tensor& s = THPVariable_Unpack(a[2]);
            if (s.scalar_type() != at::kFloat || !s.is_cuda()) raise(PyExc_ValueError, "w_scale tensor must be float32 on the GPU");
            ws_dev = static_cast<const float*>(s.data_ptr());
        } else {
            ws_host = static_cast<float>(float_arg(a[2]));
        }
        if (!codes.is_contiguous()) codes = codes.contiguous();
        const int layout = static_cast<int>(long_arg(a[5]));
        const double eps = float_arg(a[7]);
        const unsigned flags = static_cast<unsigned>(long_arg(a[9]));
        const long path = long_arg(a[10]);
        void* const stream = c10::cuda::getCurrentCUDAStream().stream();
        const int bias_type = bias ? dtype_code(bias->scalar_type()) : 0;
        const void* const bias_ptr = bias ? bias->data_ptr() : nullptr;
        const float* xs_ptr = x_scale ? static_cast<const float*>(x_scale->data_ptr()) : nullptr;
        // auto: the tensor-core contraction above decode_max_tokens tokens, and from 16 tokens on for matrices of at least 4 Mi
        // weights (measured: 4096 x 4096 at 32 tokens 14 us against 20 us on the decode kernel; small layers the reverse)
        const bool contraction = path == 2 || (path == 0 && (m > long_arg(a[12]) || (m >= 16 && n * k >= (1 << 22))));
        if (m > 0) {
            const int64_t ldy = y.stride(0);
            const int y_code = dtype_code(y.scalar_type());
            int32_t* const acc_ptr = static_cast<int32_t*>(ptr(acc));
            const uint8_t* const codes_ptr = static_cast<const uint8_t*>(codes.data_ptr());
            int rc;
            if (contraction) {
                const at::Tensor ws = contraction_workspace(m, n, k, x.options().dtype(at::kByte));
                const int x_code = dtype_code(rows.scalar_type());
                pybind11::gil_scoped_release nogil;
                rc = wf_bitlinear_prefill(rows.data_ptr(), x_code, rows.stride(0), xs_ptr, codes_ptr, layout, ws_dev, ws_host, bias_ptr, bias_type,
                                          y.data_ptr(), y_code, ldy, acc_ptr, m, n, k, static_cast<float>(eps), ws.data_ptr(),
                                          static_cast<size_t>(ws.numel()), flags, stream);
            } else {
                Quantized pre;  // alive until the launch: its memory goes back to this stream's pool
                if (rows.scalar_type() != at::kChar && (m >= long_arg(a[13]) || m * k >= long_arg(a[14])) && !wf_decode_fuses_quant(m, k, n * k, 1)) {
                    // every CTA of the decode kernel quantizes the tokens of its problem: from this many tokens on one
                    // quantization kernel in front of it is cheaper (same arithmetic, same bits), unless the launch is of
                    // the kind that does it on the way
                    pre = quantize(rows, false, eps, false, stream);
                    rows = pre.q;
                    xs_ptr = static_cast<const float*>(pre.scale.data_ptr());
                }
                const int x_code = dtype_code(rows.scalar_type());
                pybind11::gil_scoped_release nogil;
                rc = wf_bitlinear_decode(rows.data_ptr(), x_code, rows.stride(0), xs_ptr, codes_ptr, layout, ws_dev, ws_host, bias_ptr, bias_type,
                                         y.data_ptr(), y_code, ldy, acc_ptr, m, n, k, static_cast<float>(eps), flags, stream);
            }
            check(rc, contraction ? "wf_bitlinear_prefill" : "wf_bitlinear_decode");
        }
        at::Tensor shaped = y;
        if (x.dim() != 2 || y.dim() != 2 || y.size(0) != m || y.size(1) != n) {
            std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
            shape.push_back(n);
            shaped = y.reshape(shape);
        }
        return acc.defined() ? wrap_all({shaped, acc}) : wrap(shaped);
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// prompt_layers(layers, h, cos, sin, xq, aq, scale, qkv, gu, att, res, ws, B, S, n_q, n_kv, D, mode, eps, decode_max_tokens,
//               prequant_min_tokens, prequant_min_elems)
// The layers of a decoder's prompt pass (bf16, no sub-layer norms, one GPU) on the caller's buffers; `layers`: per layer a tuple of
// (qkv codes, qkv row scales, o codes, o scale, gate/up codes, gate/up row scales, down codes, down scale, norm 1, norm 2, keys, values).
// The same calls as the loop in the decoder makes, thirteen launches per layer; from Python their nine wrappers took about 100 us of
// host time per layer, which is what bounded a short prompt.  `res` holds the last layer's output of down, not yet added to h.
PyObject* prompt_layers(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    try {
        if (n_args != 22) raise(PyExc_TypeError, "prompt_layers takes 22 arguments");
        struct Layer {
            const uint8_t *qkv, *o, *gu, *down;
            const float *qkv_s, *o_s, *gu_s, *down_s;
            const void *n1, *n2;
            void *kc, *vc;
        };
        const at::Tensor &h = tensor(a[1]), &cos = tensor(a[2]), &sin = tensor(a[3]), &xq = tensor(a[4]), &aq = tensor(a[5]), &scale = tensor(a[6]), &qkv = tensor(a[7]),
                         &gu = tensor(a[8]), &att = tensor(a[9]), &res = tensor(a[10]), &ws = tensor(a[11]);
        const int64_t B = long_arg(a[12]), S = long_arg(a[13]);
        const int nq = static_cast<int>(long_arg(a[14])), nkv = static_cast<int>(long_arg(a[15])), D = static_cast<int>(long_arg(a[16]));
        const int mode = static_cast<int>(long_arg(a[17]));
        const float eps = static_cast<float>(float_arg(a[18]));
        const long decode_max = long_arg(a[19]), pre_tokens = long_arg(a[20]), pre_elems = long_arg(a[21]);
        const int64_t M = h.size(0), hidden = h.size(1), qd = static_cast<int64_t>(nq) * D, kvd = static_cast<int64_t>(nkv) * D, inter = aq.size(1);
        const auto rows_of = [&](const at::Tensor& t, int64_t width) { return t.dim() == 2 && t.size(0) == M && t.size(1) == width && t.is_contiguous(); };
        if (h.dim() != 2 || M != B * S || xq.numel() < M * std::max(hidden, qd) || scale.numel() != M || !rows_of(aq, inter) || !rows_of(qkv, qd + 2 * kvd) ||
            !rows_of(gu, 2 * inter) || !rows_of(att, qd) || !rows_of(res, hidden) || !h.is_contiguous())
            raise(PyExc_ValueError, "prompt_layers: a buffer does not have its shape");
        const auto all_of = [](at::ScalarType type, std::initializer_list<const at::Tensor*> ts) {
            return std::all_of(ts.begin(), ts.end(), [&](const at::Tensor* t) { return t->scalar_type() == type && t->is_contiguous(); });
        };
        if (B < 1 || S < 1 || nq < 1 || nkv < 1 || D < 2 || !all_of(at::kBFloat16, {&h, &qkv, &gu, &att, &res}) || !all_of(at::kChar, {&xq, &aq}) ||
            !all_of(at::kFloat, {&cos, &sin, &scale}) || !all_of(at::kByte, {&ws}) || cos.numel() < S * (D / 2) || sin.numel() < S * (D / 2))
            raise(PyExc_ValueError, "prompt_layers: a buffer does not have its type, or the rotary tables are shorter than the prompt");
        if (!PyList_Check(a[0])) raise(PyExc_TypeError, "prompt_layers: layers must be a list");
        std::vector<Layer> layers(static_cast<size_t>(PyList_GET_SIZE(a[0])));
        int64_t T = 0;
        bool together = true;  // on one device
        for (size_t i = 0; i < layers.size(); ++i) {
            PyObject* t = PyList_GET_ITEM(a[0], static_cast<Py_ssize_t>(i));
            if (!PyTuple_Check(t) || PyTuple_GET_SIZE(t) != 12) raise(PyExc_TypeError, "prompt_layers: a layer is a tuple of twelve tensors");
            const at::Tensor* e[12];
            for (int j = 0; j < 12; ++j) e[j] = &tensor(PyTuple_GET_ITEM(t, j));
            if (!all_of(at::kByte, {e[0], e[2], e[4], e[6]}) || !all_of(at::kFloat, {e[1], e[3], e[5], e[7]}) || !all_of(at::kBFloat16, {e[8], e[9], e[10], e[11]}))
                raise(PyExc_ValueError, "prompt_layers: a layer's tensor does not have its type, or is not contiguous");
            if (e[10]->dim() != 4 || (i && e[10]->size(2) != T)) raise(PyExc_ValueError, "prompt_layers: caches are [B, heads, T, D] with one T for all layers");
            T = e[10]->size(2);
            if (e[0]->numel() * 4 != (qd + 2 * kvd) * hidden || e[1]->numel() != qd + 2 * kvd || e[2]->numel() * 4 != hidden * qd || e[3]->numel() < 1 ||
                e[4]->numel() * 4 != 2 * inter * hidden || e[5]->numel() != 2 * inter || e[6]->numel() * 4 != hidden * inter || e[7]->numel() < 1 ||
                e[8]->numel() != hidden || e[9]->numel() != hidden || e[10]->numel() != B * T * kvd || e[11]->numel() != B * T * kvd || S > T)
                raise(PyExc_ValueError, "prompt_layers: a layer's tensor does not have its shape");
            for (const at::Tensor* one : e) together = together && one->device() == h.device();
            layers[i] = {static_cast<const uint8_t*>(e[0]->data_ptr()), static_cast<const uint8_t*>(e[2]->data_ptr()), static_cast<const uint8_t*>(e[4]->data_ptr()),
                         static_cast<const uint8_t*>(e[6]->data_ptr()), e[1]->data_ptr<float>(), e[3]->data_ptr<float>(), e[5]->data_ptr<float>(), e[7]->data_ptr<float>(),
                         e[8]->data_ptr(), e[9]->data_ptr(), e[10]->data_ptr(), e[11]->data_ptr()};
        }
        for (const at::Tensor* one : {&cos, &sin, &xq, &aq, &scale, &qkv, &gu, &att, &res, &ws}) together = together && one->device() == h.device();
        need_cuda({&h});
        if (!together) raise(PyExc_ValueError, "prompt_layers: tensors on different devices");
        c10::cuda::CUDAGuard guard(h.device());
        void* const stream = c10::cuda::getCurrentCUDAStream().stream();
        int8_t* const q8 = xq.data_ptr<int8_t>();
        int8_t* const a8 = aq.data_ptr<int8_t>();
        float* const xs = scale.data_ptr<float>();
        const auto bytes = h.options().dtype(at::kByte);
        const char* what = "";
        int rc = 0;
        // one projection of the tokens, by the rule of bitlinear(); from bf16 (x_scale null) or int8
        const auto project = [&](const void* x, int type, const float* x_scale, const uint8_t* codes, const float* w_scale, int64_t k) {
            if (M > decode_max || (M >= 16 && hidden * k >= (1 << 22))) {
                const at::Tensor own = contraction_workspace(M, hidden, k, bytes);
                what = "wf_bitlinear_prefill";
                return wf_bitlinear_prefill(x, type, k, x_scale, codes, WF_LAYOUT_WF16, w_scale, 0.f, nullptr, 0, res.data_ptr(), WF_BF16, hidden, nullptr, M, hidden, k, 1e-5f,
                                            own.data_ptr(), static_cast<size_t>(own.numel()), 0, stream);
            }
            if (type != WF_I8 && (M >= pre_tokens || M * k >= pre_elems) && !wf_decode_fuses_quant(M, k, hidden * k, 1)) {
                what = "wf_act_quant_i8";
                if (const int e = wf_act_quant_i8(x, type, M, k, k, WF_ACT_PER_TOKEN, 1e-5f, q8, xs, nullptr, stream)) return e;
                x = q8;
                type = WF_I8;
                x_scale = xs;
            }
            what = "wf_bitlinear_decode";
            return wf_bitlinear_decode(x, type, k, x_scale, codes, WF_LAYOUT_WF16, w_scale, 0.f, nullptr, 0, res.data_ptr(), WF_BF16, hidden, nullptr, M, hidden, k, 1e-5f, 0, stream);
        };
        {
            pybind11::gil_scoped_release nogil;
            const auto step = [&](int e, const char* name) {
                what = name;
                return e;
            };
            char* const qkv_p = static_cast<char*>(qkv.data_ptr());
            char* const gu_p = static_cast<char*>(gu.data_ptr());
            const size_t ws_bytes = static_cast<size_t>(ws.numel());
            bool first = true;
            for (const Layer& L : layers) {
                if ((rc = step(wf_add_rmsnorm_quant_bf16(h.data_ptr(), first ? nullptr : res.data_ptr(), L.n1, nullptr, q8, xs, M, hidden, eps, 1e-5f, first ? 0 : WF_FLAG_PDL, stream), "wf_add_rmsnorm_quant_bf16"))) break;
                first = false;
                if ((rc = step(wf_bitlinear_prefill_rows(q8, hidden, xs, L.qkv, L.qkv_s, qkv_p, WF_BF16, qd + 2 * kvd, M, qd + 2 * kvd, hidden, ws.data_ptr(), ws_bytes, stream), "wf_bitlinear_prefill_rows"))) break;
                if ((rc = step(wf_rope_kv_prompt_ld_bf16(qkv_p, qd + 2 * kvd, qkv_p + 2 * qd, qkv_p + 2 * (qd + kvd), qd + 2 * kvd, cos.data_ptr<float>(), sin.data_ptr<float>(), L.kc, L.vc, B, S, nq,
                                                         nkv, D, T, WF_FLAG_PDL, stream), "wf_rope_kv_prompt_bf16"))) break;
                if ((rc = step(wf_attn_prompt_bf16(qkv_p, qd + 2 * kvd, L.kc, L.vc, att.data_ptr(), B, S, nq, nkv, D, T, static_cast<float>(std::pow(static_cast<double>(D), -0.5)), WF_FLAG_PDL, stream), "wf_attn_prompt_bf16"))) break;
                if ((rc = project(att.data_ptr(), WF_BF16, nullptr, L.o, L.o_s, qd))) break;
                if ((rc = step(wf_add_rmsnorm_quant_bf16(h.data_ptr(), res.data_ptr(), L.n2, nullptr, q8, xs, M, hidden, eps, 1e-5f, WF_FLAG_PDL, stream), "wf_add_rmsnorm_quant_bf16"))) break;
                if ((rc = step(wf_bitlinear_prefill_rows(q8, hidden, xs, L.gu, L.gu_s, gu_p, WF_BF16, 2 * inter, M, 2 * inter, hidden, ws.data_ptr(), ws_bytes, stream), "wf_bitlinear_prefill_rows"))) break;
                if ((rc = step(wf_act_mul_quant_ld_bf16(gu_p, gu_p + 2 * inter, 2 * inter, nullptr, a8, xs, M, inter, mode, 1e-5f, WF_FLAG_PDL, stream), "wf_act_mul_quant_bf16"))) break;
                if ((rc = project(a8, WF_I8, xs, L.down, L.down_s, inter))) break;
            }
        }
        check(rc, what);
        Py_RETURN_NONE;
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------- 8-bit caches, weights; logits

bool half_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool float_type(at::ScalarType t) { return half_type(t) || t == at::kFloat; }
bool one_device(const at::Device& d, std::initializer_list<const at::Tensor*> ts) {
    return std::all_of(ts.begin(), ts.end(), [&](const at::Tensor* t) { return !t || t->device() == d; });
}
unsigned pdl_flag(PyObject* o) { return truth(o) ? WF_FLAG_PDL : 0; }

struct CacheI8 {
    const at::Tensor *k, *v, *ks, *vs;
    int64_t B, nkv, T, D;
    int8_t* kp() const { return static_cast<int8_t*>(k->data_ptr()); }
    int8_t* vp() const { return static_cast<int8_t*>(v->data_ptr()); }
    float* ksp() const { return static_cast<float*>(ks->data_ptr()); }
    float* vsp() const { return static_cast<float*>(vs->data_ptr()); }
};
CacheI8 cache_i8(PyObject* o, const char* name, std::initializer_list<const at::Tensor*> others) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) raise(PyExc_TypeError, message(name, " needs a KVCacheI8"));
    CacheI8 c;
    c.k = &tensor(PyTuple_GET_ITEM(o, 0));
    c.v = &tensor(PyTuple_GET_ITEM(o, 1));
    c.ks = &tensor(PyTuple_GET_ITEM(o, 2));
    c.vs = &tensor(PyTuple_GET_ITEM(o, 3));
    need_cuda({c.k, c.v, c.ks, c.vs});
    need_cuda(others);
    if (c.k->dim() != 4 || c.k->scalar_type() != at::kChar || c.v->scalar_type() != at::kChar || c.v->sizes() != c.k->sizes() || !c.k->is_contiguous() || !c.v->is_contiguous() ||
        c.ks->scalar_type() != at::kFloat || c.vs->scalar_type() != at::kFloat || c.ks->sizes() != c.k->sizes().slice(0, 3) || c.vs->sizes() != c.k->sizes().slice(0, 3) ||
        !c.ks->is_contiguous() || !c.vs->is_contiguous())
        raise(PyExc_ValueError, message(name, " needs contiguous int8 caches [B, nkv, T, D] of one shape and contiguous float32 scales [B, nkv, T]"));
    if (!one_device(c.k->device(), {c.v, c.ks, c.vs}) || !one_device(c.k->device(), others)) raise(PyExc_ValueError, message(name, " needs its tensors on one device"));
    c.B = c.k->size(0); c.nkv = c.k->size(1); c.T = c.k->size(2); c.D = c.k->size(3);
    return c;
}
// address and stride of a position for all sequences or one for each
std::pair<const int64_t*, int> positions(const at::Tensor* pos, int64_t B, const char* name) {
    if (!pos) return {nullptr, 0};
    const bool one = pos->numel() == 1;
    if (pos->scalar_type() != at::kLong || !(one || (pos->dim() == 1 && pos->size(0) == B && pos->stride(0) == 1)))
        raise(PyExc_ValueError, message(name, " needs int64 positions: a scalar, or one for each of the ", B, " sequences with unit stride; got ", pos->scalar_type(), " ", pos->sizes()));
    return {static_cast<const int64_t*>(pos->data_ptr()), one ? 0 : 1};
}
// Elements of each of the `rows` rows that t is: of shape [rows, width], or contiguous with the rows in its leading dimensions (one at least, unless t is a single
// row) and behind them a width, heads of D, groups of heads for each of nkv, each with ones wherever.  A number of rows that is another one is never taken for heads.
int64_t row_width(const at::Tensor& t, int64_t rows, int64_t nkv, int64_t D, const char* name) {
    const auto dims = t.sizes();
    if (dims.size() == 2) {
        if (dims[0] == rows) return dims[1];
    } else if (t.is_contiguous() && !dims.empty()) {
        size_t i = 0;
        int64_t front = 1;
        if (dims.size() > 2 || rows != 1)
            for (front = dims[i++]; front != rows && i < dims.size(); ++i) front *= dims[i];
        std::vector<int64_t> rest;
        for (; i < dims.size(); ++i)
            if (dims[i] != 1) rest.push_back(dims[i]);
        const bool heads = rest.size() <= 1 || (rest.size() == 2 && (rest[1] == D || rest[0] == nkv)) || (rest.size() == 3 && rest[0] == nkv && rest[2] == D);
        if (front == rows && heads) return t.numel() / rows;
    }
    raise(PyExc_ValueError, message(name, " must have ", rows, " row(s), as the cache and the number of new tokens say, two-dimensional or contiguous; got ", t.sizes(), " with strides ", t.strides()));
}
// elements from one row of `width` to the next: contiguous in any shape, or two-dimensional with unit inner stride
int64_t row_stride(const at::Tensor& t, int64_t rows, int64_t width, int64_t nkv, int64_t D, const char* name, at::ScalarType type) {
    if (t.scalar_type() == type && row_width(t, rows, nkv, D, name) == width) {
        if (t.is_contiguous()) return width;
        if (t.dim() == 2 && t.stride(1) == 1 && (t.stride(0) >= width || rows == 1)) return std::max(t.stride(0), width);
    }
    raise(PyExc_ValueError, message(name, " must be ", type, " rows [", rows, ", ", width, "], contiguous or two-dimensional with unit inner stride; got ", t.scalar_type(), " ", t.sizes(),
                                     " with strides ", t.strides()));
}

// rope_kv_i8(q, k, v, cos, sin, pos, cache, s, out, pdl) -> out
PyObject* rope_kv_i8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    try {
        if (n_args != 10) raise(PyExc_TypeError, "rope_kv_i8 takes 10 arguments");
        const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &cos = tensor(a[3]), &sin = tensor(a[4]), &pos = tensor(a[5]);
        const at::Tensor* given = optional_tensor(a[8]);
        const CacheI8 c = cache_i8(a[6], "rope_kv_i8_", {&q, &k, &v, &cos, &sin, &pos, given});
        const int64_t s = long_arg(a[7]);
        const at::Tensor& out = given ? *given : q;
        if (s < 0 || s > INT32_MAX || !half_type(q.scalar_type())) raise(PyExc_ValueError, message("rope_kv_i8_ needs bf16 or f16 tensors and s of 0 to 2^31 - 1, got ", q.scalar_type(), " and ", s));
        if (c.B && s) {
            const int64_t rows = c.B * s, heads = row_width(q, rows, c.nkv, c.D, "q") / std::max<int64_t>(c.D, 1);
            for (const at::Tensor* t : {&cos, &sin})
                if (t->scalar_type() != at::kFloat || t->dim() < 2 || t->size(-1) != c.D / 2 || t->numel() < c.T * (c.D / 2) || !t->is_contiguous())
                    raise(PyExc_ValueError, message("rope_kv_i8_ needs contiguous float32 rotary tables [T, D/2] = [", c.T, ", ", c.D / 2, "] or longer; got ", t->scalar_type(), " ", t->sizes()));
            const auto stride = [&](const at::Tensor& t, int64_t n, const char* name) { return row_stride(t, rows, n * c.D, c.nkv, c.D, name, q.scalar_type()); };
            const int64_t ldq = stride(q, heads, "q"), ldo = stride(out, heads, "out"), ldk = stride(k, c.nkv, "k"), ldv = stride(v, c.nkv, "v");
            if (ldk != ldv) raise(PyExc_ValueError, message("k and v must have the same row stride, got ", ldk, " and ", ldv));
            const auto at = positions(&pos, c.B, "rope_kv_i8_");
            const unsigned flags = pdl_flag(a[9]);
            c10::cuda::CUDAGuard guard(q.device());
            check(wf_rope_kv_i8(q.data_ptr(), ldq, k.data_ptr(), v.data_ptr(), ldk, dtype_code(q.scalar_type()), static_cast<const float*>(cos.data_ptr()),
                                static_cast<const float*>(sin.data_ptr()), at.first, at.second, out.data_ptr(), ldo, c.kp(), c.vp(), c.ksp(), c.vsp(), c.B, s,
                                static_cast<int>(heads), static_cast<int>(c.nkv), static_cast<int>(c.D), c.T, flags, c10::cuda::getCurrentCUDAStream().stream()),
                  "wf_rope_kv_i8");
        }
        return wrap(out);
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// kv_read_i8(cache, s, start, dtype, pdl) -> (k, v)
PyObject* kv_read_i8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    try {
        if (n_args != 5) raise(PyExc_TypeError, "kv_read_i8 takes 5 arguments");
        const CacheI8 c = cache_i8(a[0], "kv_read_i8", {});
        const int64_t s = long_arg(a[1]), start = long_arg(a[2]);
        if (!THPDtype_Check(a[3])) raise(PyExc_TypeError, "dtype must be a torch.dtype");
        const at::ScalarType type = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
        if (!half_type(type) || s < 0 || start < 0 || start > c.T - s)
            raise(PyExc_ValueError, message("kv_read_i8 reads positions of 0 .. ", c.T, " as bf16 or f16; got ", s, " from ", start, " on as ", type));
        const unsigned flags = pdl_flag(a[4]);
        c10::cuda::CUDAGuard guard(c.k->device());
        const at::Tensor k = at::empty({c.B, c.nkv, s, c.D}, c.k->options().dtype(type)), v = at::empty({c.B, c.nkv, s, c.D}, c.k->options().dtype(type));
        if (k.numel())
            check(wf_kv_read_i8(c.kp(), c.vp(), c.ksp(), c.vsp(), k.data_ptr(), v.data_ptr(), dtype_code(type), c.B * c.nkv, c.T, start, s, static_cast<int>(c.D), flags,
                                c10::cuda::getCurrentCUDAStream().stream()),
                  "wf_kv_read_i8");
        return wrap_all({k, v});
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// Workspaces of attn_decode_i8 calls that bring none, by device and stream: launches of one stream run one after the other, and the memory goes back to
// that stream.  A captured call gets one of the graph's own, cleared on every replay.  A stream that is not torch's own (its id is its handle) gets one for the
// call: when such a stream is destroyed another may have its handle.  The per-thread default stream has one handle for a stream in every thread, which the
// allocator does not know either: there the workspace is the caller's.  (Never destroyed: the process's end does not wait for this library.)
constexpr size_t KEPT_WORKSPACES = 16;
struct KeptWorkspace {
    int device;
    void* stream;
    at::Tensor ws;
};
at::Tensor stream_workspace(int64_t bytes, const at::Tensor& like, const c10::cuda::CUDAStream& current) {
    static std::vector<KeptWorkspace>& kept = *new std::vector<KeptWorkspace>();
    const auto options = like.options().dtype(at::kByte);
    void* const stream = current.stream();
    if (stream == cudaStreamPerThread) raise(PyExc_ValueError, "attn_decode_i8 needs a workspace of the caller's on the per-thread default stream");
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return at::zeros({bytes}, options);
    if (stream && current.id() == static_cast<c10::StreamId>(reinterpret_cast<intptr_t>(stream))) return at::zeros({bytes}, options);
    const int device = like.device().index();
    for (size_t i = 0; i < kept.size(); ++i)
        if (kept[i].device == device && kept[i].stream == stream) {
            if (kept[i].ws.numel() >= bytes) return kept[i].ws;
            kept.erase(kept.begin() + static_cast<std::ptrdiff_t>(i));
            break;
        }
    if (kept.size() >= KEPT_WORKSPACES) kept.erase(kept.begin());
    kept.push_back({device, stream, at::zeros({bytes}, options)});
    return kept.back().ws;
}

// attn_decode_i8(q, cache, pos, out, scale, pdl, workspace) -> out
PyObject* attn_decode_i8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    try {
        if (n_args != 7) raise(PyExc_TypeError, "attn_decode_i8 takes 7 arguments");
        const at::Tensor& q = tensor(a[0]);
        const at::Tensor *pos = optional_tensor(a[2]), *given = optional_tensor(a[3]), *workspace = optional_tensor(a[6]);
        const CacheI8 c = cache_i8(a[1], "attn_decode_i8", {&q, pos, given, workspace});
        if (!half_type(q.scalar_type()) || q.dim() < 1 || c.D < 1)
            raise(PyExc_ValueError, message("attn_decode_i8 needs bf16 or f16 queries [B, nq*D], got ", q.scalar_type(), " ", q.sizes()));
        const int64_t nq = (c.B ? row_width(q, c.B, c.nkv, c.D, "q") : q.size(-1)) / c.D;
        if (given && (given->scalar_type() != q.scalar_type() || given->numel() != q.numel() || !given->is_contiguous()))
            raise(PyExc_ValueError, "attn_decode_i8 needs a contiguous output of the type and size of q");
        if (workspace && (workspace->element_size() != 1 || !workspace->is_contiguous())) raise(PyExc_ValueError, "attn_decode_i8 needs a workspace of contiguous bytes");
        const double scale = a[4] == Py_None ? std::pow(static_cast<double>(c.D), -0.5) : float_arg(a[4]);
        const unsigned flags = pdl_flag(a[5]);
        c10::cuda::CUDAGuard guard(q.device());
        const at::Tensor out = given ? *given : at::empty({c.B, nq * c.D}, q.options());
        if (c.B) {
            const auto at = positions(pos, c.B, "attn_decode_i8");
            const int64_t ldq = row_stride(q, c.B, nq * c.D, c.nkv, c.D, "q", q.scalar_type());
            const auto from = reinterpret_cast<uintptr_t>(q.data_ptr()), to = reinterpret_cast<uintptr_t>(out.data_ptr());
            if (to < from + 2 * ((c.B - 1) * ldq + nq * c.D) && from < to + 2 * c.B * nq * c.D)
                raise(PyExc_ValueError, "attn_decode_i8 cannot write over q: parts of a sequence that run later still read it");
            const c10::cuda::CUDAStream current = c10::cuda::getCurrentCUDAStream();
            const at::Tensor ws = workspace ? *workspace
                                            : stream_workspace(static_cast<int64_t>(std::max<size_t>(wf_attn_decode_i8_workspace_bytes(static_cast<int>(nq), static_cast<int>(c.nkv), static_cast<int>(c.D)), 1)), q, current);
            check(wf_attn_decode_i8(q.data_ptr(), dtype_code(q.scalar_type()), ldq, c.kp(), c.vp(), c.ksp(), c.vsp(), at.first, at.second, out.data_ptr(), c.B,
                                    static_cast<int>(nq), static_cast<int>(c.nkv), static_cast<int>(c.D), c.T, static_cast<float>(scale), ws.data_ptr(),
                                    static_cast<size_t>(ws.numel()), flags, current.stream()),
                  "wf_attn_decode_i8");
        }
        return wrap(out);
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// linear_i8(x, codes, w_scale, x_scale, bias, out, out_dtype, pdl) -> y
PyObject* linear_i8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    try {
        if (n_args != 8) raise(PyExc_TypeError, "linear_i8 takes 8 arguments");
        const at::Tensor &x = tensor(a[0]), &codes = tensor(a[1]), &w_scale = tensor(a[2]);
        const at::Tensor *x_scale = optional_tensor(a[3]), *bias = optional_tensor(a[4]), *out = optional_tensor(a[5]);
        need_cuda({&x, &codes, &w_scale, x_scale, bias, out});
        if (x.dim() < 1 || codes.dim() != 2 || codes.scalar_type() != at::kChar || codes.size(1) != x.size(-1) || codes.size(1) < 1 || codes.size(0) < 1)
            raise(PyExc_ValueError, message("linear_i8 needs int8 codes [N, K] for x [..., K], got ", codes.scalar_type(), " ", codes.sizes(), " and ", x.sizes()));
        const int64_t n = codes.size(0), k = codes.size(1), padded = (k + 15) / 16 * 16;
        if (k > 1 && codes.stride(1) != 1) raise(PyExc_ValueError, "linear_i8 needs codes with unit inner stride");
        if (w_scale.scalar_type() != at::kFloat || w_scale.dim() != 1 || w_scale.size(0) != n || !w_scale.is_contiguous()) raise(PyExc_ValueError, "linear_i8 needs a contiguous float32 w_scale [N]");
        if (bias && (bias->dim() != 1 || bias->size(0) != n || !bias->is_contiguous() || !float_type(bias->scalar_type())))
            raise(PyExc_ValueError, "linear_i8 needs a contiguous bias [N] of float32, bf16 or f16");
        if (!one_device(x.device(), {&codes, &w_scale, x_scale, bias, out})) raise(PyExc_ValueError, "linear_i8 needs its tensors on one device");
        at::Tensor rows = x.dim() == 2 ? x : x.reshape({-1, k});
        const int64_t m = rows.size(0);
        const bool coded = x.scalar_type() == at::kChar;
        if (coded) {
            if (!x_scale || x_scale->scalar_type() != at::kFloat || x_scale->numel() != m || !x_scale->is_contiguous())
                raise(PyExc_ValueError, "linear_i8 needs a contiguous float32 x_scale of one element per token beside int8 tokens");
        } else if (!float_type(x.scalar_type()) || x_scale) {
            raise(PyExc_ValueError, message("linear_i8 takes tokens of float32, bf16, f16, or int8 with x_scale; got ", x.scalar_type(), x_scale ? " with x_scale" : ""));
        }
        at::ScalarType type = coded ? at::kBFloat16 : x.scalar_type();
        if (a[6] != Py_None) {
            if (!THPDtype_Check(a[6])) raise(PyExc_TypeError, "out_dtype must be a torch.dtype");
            type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
        }
        const unsigned flags = pdl_flag(a[7]);
        c10::cuda::CUDAGuard guard(x.device());
        at::Tensor y;
        if (out) {
            y = *out;
        } else {
            if (!float_type(type)) raise(PyExc_ValueError, "linear_i8: the output is bf16, f16 or float32");
            std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
            shape.push_back(n);
            y = at::empty(shape, x.options().dtype(type));
        }
        if (y.dim() != 2 && (y.dim() < 1 || y.size(-1) != n || y.numel() != m * n || !y.is_contiguous()))
            raise(PyExc_ValueError, "linear_i8: `out` must be [..., N], contiguous or two-dimensional");
        const at::Tensor y2 = y.dim() == 2 ? y : y.view({m, n});
        if (y2.size(0) != m || y2.size(1) != n || (n > 1 && y2.stride(1) != 1) || !float_type(y.scalar_type()) || (m > 1 && y2.stride(0) < n))
            raise(PyExc_ValueError, "linear_i8: `out` must be [..., N] of bf16, f16 or float32 with unit inner stride");
        if (m) {
            if ((k > 1 && rows.stride(1) != 1) || (m > 1 && rows.stride(0) < k)) rows = rows.contiguous();
            void* const stream = c10::cuda::getCurrentCUDAStream().stream();
            const int8_t* xq = static_cast<const int8_t*>(coded ? rows.data_ptr() : nullptr);
            const float* xs = coded ? static_cast<const float*>(x_scale->data_ptr()) : nullptr;
            int64_t ldx = m > 1 ? rows.stride(0) : padded;
            unsigned how = flags;
            at::Tensor room;  // alive until the launches: its memory goes back to this stream's pool
            if (!coded) {
                const int64_t steps = (m * 4 + 15) / 16 * 16;
                room = at::empty({steps + m * padded}, x.options().dtype(at::kByte));
                float* const s = static_cast<float*>(room.data_ptr());
                int8_t* const q = static_cast<int8_t*>(room.data_ptr()) + steps;
                check(wf_quantize_rows_i8(rows.data_ptr(), dtype_code(x.scalar_type()), m > 1 ? rows.stride(0) : k, q, padded, s, m, k, WF_FLAG_PDL, stream), "wf_quantize_rows_i8");
                xq = q;
                xs = s;
                ldx = padded;
                how = WF_FLAG_PDL;  // the product asks for its first weights while the tokens are quantized
            }
            check(wf_linear_i8(xq, ldx, xs, static_cast<const int8_t*>(codes.data_ptr()), n > 1 ? codes.stride(0) : padded, static_cast<const float*>(w_scale.data_ptr()),
                               bias ? bias->data_ptr() : nullptr, bias ? dtype_code(bias->scalar_type()) : 0, y2.data_ptr(), dtype_code(y.scalar_type()), m > 1 ? y2.stride(0) : n, m, n, k, how,
                               stream),
                  "wf_linear_i8");
        }
        return wrap(y);
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// token_logprobs(logits [..., V], tokens [...], top, kept) -> (logprob, entropy, top_logprob, top_id), each [...] or [..., top]; with `kept` (a gradient will be
// taken) also the logits as rows, the tokens as a row of them and the rows' statistics
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    try {
        if (n_args != 4) raise(PyExc_TypeError, "token_logprobs takes 4 arguments");
        const at::Tensor &logits = tensor(a[0]), &given = tensor(a[1]);
        need_cuda({&logits, &given});
        const int64_t top = long_arg(a[2]);
        const bool kept = truth(a[3]);
        if (!float_type(logits.scalar_type()) || logits.dim() < 1 || logits.size(-1) < 1)
            raise(PyExc_ValueError, message("token_logprobs needs logits [..., V] of float32, bf16 or f16, got ", logits.scalar_type(), " ", logits.sizes()));
        if (given.scalar_type() != at::kLong || given.sizes() != logits.sizes().slice(0, logits.dim() - 1) || given.device() != logits.device())
            raise(PyExc_ValueError, message("token_logprobs needs int64 tokens ", logits.sizes().slice(0, logits.dim() - 1), " on the logits' device, got ", given.scalar_type(), " ", given.sizes()));
        if (logits._fw_grad(0).defined()) raise(PyExc_NotImplementedError, "token_logprobs has no forward-mode derivative");
        if (top < 0 || top > 32) raise(PyExc_ValueError, message("token_logprobs finds 0 to 32 alternatives, asked for ", top));
        c10::cuda::CUDAGuard guard(logits.device());
        const int64_t v = logits.size(-1);
        at::Tensor rows = logits.dim() == 2 ? logits : logits.reshape({-1, v});
        const int64_t r = rows.size(0);
        if ((v > 1 && rows.stride(1) != 1) || (r > 1 && rows.stride(0) < v)) rows = rows.contiguous();
        const at::Tensor tokens = given.is_contiguous() ? given : given.contiguous();
        std::vector<int64_t> shape(logits.sizes().begin(), logits.sizes().end() - 1);
        const auto f32 = logits.options().dtype(at::kFloat);
        const at::Tensor logprob = at::empty(shape, f32), entropy = at::empty(shape, f32);
        shape.push_back(top);
        const at::Tensor top_logprob = at::empty(shape, f32), top_id = at::empty(shape, f32.dtype(at::kLong));
        at::Tensor stats;
        if (kept) stats = at::empty({r, 2}, f32);
        if (r)
            check(wf_token_logprobs(rows.data_ptr(), dtype_code(rows.scalar_type()), std::max(rows.stride(0), v), static_cast<const int64_t*>(tokens.data_ptr()),
                                    static_cast<float*>(logprob.data_ptr()), static_cast<float*>(entropy.data_ptr()), kept ? static_cast<float*>(stats.data_ptr()) : nullptr,
                                    top ? static_cast<float*>(top_logprob.data_ptr()) : nullptr, top ? static_cast<int64_t*>(top_id.data_ptr()) : nullptr, static_cast<int>(top), r, v,
                                    WF_FLAG_PDL, c10::cuda::getCurrentCUDAStream().stream()),
                  "wf_token_logprobs");
        return kept ? wrap_all({logprob, entropy, top_logprob, top_id, rows, tokens, stats}) : wrap_all({logprob, entropy, top_logprob, top_id});
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// token_logprobs_grad(rows, tokens, stats, entropy, top_id, g_logprob, g_entropy, g_top) -> gradient of the rows [R, V]; the first five as token_logprobs kept or
// returned them, the others None or of their shapes
PyObject* token_logprobs_grad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    try {
        if (n_args != 8) raise(PyExc_TypeError, "token_logprobs_grad takes 8 arguments");
        const at::Tensor &rows = tensor(a[0]), &tokens = tensor(a[1]), &stats = tensor(a[2]), &entropy = tensor(a[3]), &top_id = tensor(a[4]);
        const int64_t r = rows.size(0), v = rows.size(1), top = top_id.size(-1);
        at::Tensor g[3];
        const float* gp[3] = {nullptr, nullptr, nullptr};
        for (int i = 0; i < 3; ++i) {
            const at::Tensor* t = optional_tensor(a[5 + i]);
            if (!t || !t->numel()) continue;
            need_cuda({t});
            g[i] = t->scalar_type() == at::kFloat && t->is_contiguous() ? *t : t->to(at::kFloat).contiguous();
            gp[i] = static_cast<const float*>(g[i].data_ptr());
        }
        c10::cuda::CUDAGuard guard(rows.device());
        const at::Tensor dx = at::empty({r, v}, rows.options());
        if (r)
            check(wf_token_logprobs_grad(rows.data_ptr(), dtype_code(rows.scalar_type()), std::max(rows.stride(0), v), static_cast<const int64_t*>(tokens.data_ptr()),
                                         static_cast<const float*>(stats.data_ptr()), static_cast<const float*>(entropy.data_ptr()),
                                         top ? static_cast<const int64_t*>(top_id.data_ptr()) : nullptr, static_cast<int>(top), gp[0], gp[1], gp[2], dx.data_ptr(), r, v, WF_FLAG_PDL,
                                         c10::cuda::getCurrentCUDAStream().stream()),
                  "wf_token_logprobs_grad");
        return wrap(dx);
    } catch (const PyFailure&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"rope_kv_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope_kv_i8)), METH_FASTCALL, nullptr},
    {"kv_read_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv_read_i8)), METH_FASTCALL, nullptr},
    {"attn_decode_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attn_decode_i8)), METH_FASTCALL, nullptr},
    {"linear_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_i8)), METH_FASTCALL, nullptr},
    {"token_logprobs_grad", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(token_logprobs_grad)), METH_FASTCALL, nullptr},
    {"token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(token_logprobs)), METH_FASTCALL, nullptr},
    {"prompt_layers", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prompt_layers)), METH_FASTCALL, nullptr},
    {"act_quant_i8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(act_quant_i8)), METH_FASTCALL, nullptr},
    {"bitlinear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bitlinear)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "wf_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_wf_host() {
    PyObject* m = PyModule_Create(&module);
    // the tensors it takes and returns are torch's C++ objects: the loader compares this with the torch that is running
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) Py_CLEAR(m);
    return m;
}
