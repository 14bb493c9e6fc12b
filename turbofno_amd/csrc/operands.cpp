// Python extension `_operands`: the operand checks of the binding (turbofno_amd/api.py) and the two layer calls without a trip
// through Python per tensor attribute. A call through the ctypes binding spent 6.7 us on the host, 2.5 of them on checks and
// conversions in Python, for kernels of 5 us; through this module it spends 3.5 (S = 1, K = 8, N = 64, DY = 128, call after call:
// 6.84 -> 4.91 us).
//
// Nothing here decides that a call is wrong: whatever does not pass is handed back (None, or -1) and takes the checks in Python,
// which raise. Only plain torch.Tensor / Parameter objects are looked at, so subclasses and wrappers keep their own behaviour, and
// nothing is kept from one call to the next.
#include "../../include/turbofno.h"
#include "places.h"
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <climits>
#include <vector>

namespace {

using Layer1d = int (*)(int, int, int, int, int, const void*, const void*, void*, float, float, void*);
using Layer2d = int (*)(int, int, int, int, int, const void*, const void*, void*, float, float, void*, size_t, int, void*);

// a contiguous tensor of that type on a GPU; the device is the one that `device` names, or becomes it if that is negative
const at::Tensor* gpu_tensor(PyObject* o, at::ScalarType type, int& device)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.scalar_type() != type || !t.is_contiguous()) return nullptr;
    if (device < 0) device = t.get_device();
    return t.get_device() == device ? &t : nullptr;
}

// The interpreter's lock is given back while a launch waits for room in the queue (the caller's frame holds the operands), and taken again
// however the call ends
struct WithoutLock {
    PyThreadState* held = PyEval_SaveThread();
    ~WithoutLock() { PyEval_RestoreThread(held); }
};

bool fits_int(int64_t v) { return v >= 0 && v <= INT_MAX; }

// alpha as anything with a complex value; false leaves the question to Python
bool complex_value(PyObject* o, float& re, float& im)
{
    const Py_complex v = PyComplex_AsCComplex(o);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    re = (float)v.real;
    im = (float)v.imag;
    return true;
}
bool integer_value(PyObject* o, long long& v)
{
    if (!PyLong_Check(o)) return false;
    v = PyLong_AsLongLong(o);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
void* pointer_value(PyObject* o, bool& ok)
{
    void* p = PyLong_Check(o) ? PyLong_AsVoidPtr(o) : nullptr;
    ok = PyLong_Check(o) && !PyErr_Occurred();
    PyErr_Clear();
    return p;
}

// operands(t0, n0, t1, n1, ...): the addresses of contiguous complex64 tensors of exactly n elements each, all on one GPU, else None
PyObject* operands(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    if (count < 2 || count % 2 || count > 8) Py_RETURN_NONE;
    const void* address[4];
    int device = -1;
    try {
        for (Py_ssize_t i = 0; i < count; i += 2) {
            const at::Tensor* t = gpu_tensor(args[i], at::kComplexFloat, device);
            long long n;
            if (!t || !integer_value(args[i + 1], n) || t->numel() != n) Py_RETURN_NONE;
            address[i / 2] = t->data_ptr();
        }
    } catch (...) {
        Py_RETURN_NONE;
    }
    PyObject* tuple = PyTuple_New(count / 2);
    if (!tuple) return nullptr;
    for (Py_ssize_t i = 0; i < count / 2; ++i) PyTuple_SET_ITEM(tuple, i, PyLong_FromVoidPtr(const_cast<void*>(address[i])));
    return tuple;
}

// layer_1d(function, x, W, y, alpha, dimX, stream): the status of turbofno_layer_1d, -1 if the operands are for Python to judge
PyObject* layer_1d(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int rc = -1;
    if (count == 7) {
        try {
            int device = -1;
            bool ok_f, ok_s;
            const auto call = reinterpret_cast<Layer1d>(pointer_value(args[0], ok_f));
            void* stream = pointer_value(args[6], ok_s);
            const at::Tensor *x = gpu_tensor(args[1], at::kComplexFloat, device), *W = gpu_tensor(args[2], at::kComplexFloat, device),
                             *y = gpu_tensor(args[3], at::kComplexFloat, device);
            float re, im;
            long long dimX;
            if (ok_f && call && ok_s && x && W && y && complex_value(args[4], re, im) && integer_value(args[5], dimX) &&
                x->dim() == 3 && W->dim() == 2 && y->dim() == 3) {
                const int64_t K = x->size(0), S = x->size(1), DY = x->size(2), N = W->size(0);
                if (W->size(1) == K && y->size(0) == N && y->size(1) == S && y->size(2) == DY && dimX > 0 && S % dimX == 0 &&
                    fits_int(K) && fits_int(S) && fits_int(DY) && fits_int(N) && fits_int(dimX)) {
                    void *px = x->data_ptr(), *pW = W->data_ptr(), *py = y->data_ptr();
                    const WithoutLock unlocked;
                    rc = call((int)(S / dimX), (int)dimX, (int)DY, (int)K, (int)N, px, pW, py, re, im, stream);
                }
            }
        } catch (...) {
            rc = -1;
        }
    }
    return PyLong_FromLong(rc);
}

// layer_2d(function, x, W, y, alpha, workspace, algo, stream): likewise for turbofno_layer_2d
PyObject* layer_2d(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int rc = -1;
    if (count == 8) {
        try {
            int device = -1;
            bool ok_f, ok_s;
            const auto call = reinterpret_cast<Layer2d>(pointer_value(args[0], ok_f));
            void* stream = pointer_value(args[7], ok_s);
            const at::Tensor *x = gpu_tensor(args[1], at::kComplexFloat, device), *W = gpu_tensor(args[2], at::kComplexFloat, device),
                             *y = gpu_tensor(args[3], at::kComplexFloat, device), *ws = gpu_tensor(args[5], at::kByte, device);
            float re, im;
            long long algo;
            if (ok_f && call && ok_s && x && W && y && ws && complex_value(args[4], re, im) && integer_value(args[6], algo) &&
                fits_int(algo) && x->dim() == 4 && W->dim() == 2 && y->dim() == 4) {
                const int64_t K = x->size(0), bs = x->size(1), DX = x->size(2), DY = x->size(3), N = W->size(0);
                if (W->size(1) == K && y->size(0) == N && y->size(1) == bs && y->size(2) == DX && y->size(3) == DY && fits_int(K) && fits_int(bs) &&
                    fits_int(DX) && fits_int(DY) && fits_int(N)) {
                    void *px = x->data_ptr(), *pW = W->data_ptr(), *py = y->data_ptr(), *pws = ws->data_ptr();
                    const size_t bytes = (size_t)ws->numel();
                    const WithoutLock unlocked;
                    rc = call((int)bs, (int)DX, (int)DY, (int)K, (int)N, px, pW, py, re, im, pws, bytes, (int)algo, stream);
                }
            }
        } catch (...) {
            rc = -1;
        }
    }
    return PyLong_FromLong(rc);
}

// ---- the operators around the layer (turbofno_amd/operators.py): the same checks as there, in the same order of trust: whatever does not pass is
// handed back as -1 ----

using Mix = decltype(&turbofno_mix);
using Mix8bit = decltype(&turbofno_mix_8bit);
using InputGrad = decltype(&turbofno_mix_input_grad);
using WeightGrad = decltype(&turbofno_mix_weight_grad);
using WeightGradBytes = decltype(&turbofno_mix_weight_grad_workspace_bytes);
using Norm = decltype(&turbofno_rms_norm);
using NormGrad = decltype(&turbofno_rms_norm_backward);
using NormGradBytes = decltype(&turbofno_rms_norm_backward_workspace_bytes);
using Clip = decltype(&turbofno_clip_grad_norm);
using ClipBytes = decltype(&turbofno_clip_grad_norm_workspace_bytes);
using Dropout = decltype(&turbofno_dropout);
using LayerNorm = decltype(&turbofno_layer_norm);
using LayerNorm8bit = decltype(&turbofno_layer_norm_8bit);
using LayerNormGrad = decltype(&turbofno_layer_norm_backward);
using LayerNormGradBytes = decltype(&turbofno_layer_norm_backward_workspace_bytes);
using Quantise = decltype(&turbofno_quantise_8bit);
using Mix8bitBlocks = decltype(&turbofno_mix_8bit_blocks);

struct NotHere { };                                     // an operand for Python to judge

int type_of(const at::Tensor& t)
{
    switch (t.scalar_type()) {
    case at::kComplexFloat: return TURBOFNO_C64;
    case at::kFloat: return TURBOFNO_F32;
    case at::kBFloat16: return TURBOFNO_BF16;
    default: throw NotHere();
    }
}
// a tensor of that type on that GPU whose memory holds its values
const at::Tensor& on_gpu(PyObject* o, at::ScalarType type, int device)
{
    if (!THPVariable_CheckExact(o)) throw NotHere();
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.scalar_type() != type || t.get_device() != device || t.is_conj() || t.is_neg()) throw NotHere();
    return t;
}
const at::Tensor& first_operand(PyObject* o, int device)
{
    if (!THPVariable_CheckExact(o)) throw NotHere();
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.dim() < 2 || t.size(0) <= 0) throw NotHere();
    return on_gpu(o, t.scalar_type(), device);
}
struct Field {
    void* data = nullptr;
    long ld = 0;
};
// distance between channels; the dimensions after the first have to lie side by side
long spread(const at::Tensor& t, long parts = 1)
{
    int64_t step = 1;
    for (int64_t i = t.dim() - 1; i > 0; --i) {
        if (t.size(i) != 1 && t.stride(i) != step) throw NotHere();
        step *= t.size(i);
    }
    const int64_t ld = t.size(0) > 1 ? t.stride(0) : step;
    if (ld % parts) throw NotHere();
    return ld / parts;
}
// a field of `channels` channels with the positions of `like` (whose last dimension is (re, im) where `like_pairs`), with a last dimension of two where `pairs`
Field field(PyObject* o, at::ScalarType type, int device, int64_t channels, const at::Tensor& like, bool pairs = false, bool like_pairs = false, bool optional = false)
{
    if (optional && o == Py_None) return {};
    const at::Tensor& t = on_gpu(o, type, device);
    const int64_t dims = like.dim() - (like_pairs ? 1 : 0);
    if (t.dim() != dims + (pairs ? 1 : 0) || t.size(0) != channels || (pairs && t.size(dims) != 2)) throw NotHere();
    for (int64_t i = 1; i < dims; ++i)
        if (t.size(i) != like.size(i)) throw NotHere();
    return { t.data_ptr(), spread(t, pairs ? 2 : 1) };
}
// a contiguous tensor of those sizes
void* packed(PyObject* o, at::ScalarType type, int device, std::initializer_list<int64_t> sizes, bool optional = false)
{
    if (optional && o == Py_None) return nullptr;
    const at::Tensor& t = on_gpu(o, type, device);
    if (!t.is_contiguous() || t.sizes() != at::IntArrayRef(sizes)) throw NotHere();
    return t.data_ptr();
}
// one value per position of `like`
void* per_position(PyObject* o, int device, const at::Tensor& like, bool like_pairs = false)
{
    const at::Tensor& t = on_gpu(o, at::kFloat, device);
    const int64_t dims = like.dim() - (like_pairs ? 1 : 0);
    if (!t.is_contiguous() || t.dim() != dims - 1) throw NotHere();
    for (int64_t i = 1; i < dims; ++i)
        if (t.size(i - 1) != like.size(i)) throw NotHere();
    return t.data_ptr();
}
long positions(const at::Tensor& t, bool pairs = false) { return t.numel() / t.size(0) / (pairs ? 2 : 1); }
int channels(int64_t n)
{
    if (n <= 0 || !fits_int(n)) throw NotHere();
    return (int)n;
}
template <typename F> F function(PyObject* o)
{
    bool ok;
    void* p = pointer_value(o, ok);
    if (!ok || !p) throw NotHere();
    return reinterpret_cast<F>(p);
}
int small(PyObject* o)
{
    long long v;
    if (!integer_value(o, v) || !fits_int(v)) throw NotHere();
    return (int)v;
}
void* stream_of(PyObject* o)
{
    bool ok;
    void* p = pointer_value(o, ok);
    if (!ok) throw NotHere();
    return p;
}
float real_value(PyObject* o)
{
    const double v = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) throw NotHere();
    return (float)v;
}
double double_value(PyObject* o)
{
    const double v = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) throw NotHere();
    return v;
}
// seed and offset; none without dropout
const void* seed_and_offset(PyObject* o, int device) { return packed(o, at::kLong, device, { 2 }, true); }
// the 32-bit type of values that accompany a field
at::ScalarType wide(at::ScalarType dt) { return dt == at::kComplexFloat ? dt : at::kFloat; }
// one value per position of `like`, of a type
void* at_positions(PyObject* o, at::ScalarType type, int device, const at::Tensor& like)
{
    const at::Tensor& t = on_gpu(o, type, device);
    if (!t.is_contiguous() || t.sizes() != like.sizes().slice(1)) throw NotHere();
    return t.data_ptr();
}
// one float per block of 128 channels and position of `like`
float* block_scales(PyObject* o, int device, int K, const at::Tensor& like, bool like_pairs = false)
{
    const at::Tensor& t = on_gpu(o, at::kFloat, device);
    const int64_t dims = like.dim() - (like_pairs ? 1 : 0);
    if (!t.is_contiguous() || t.dim() != dims || t.size(0) != (K + 127) / 128) throw NotHere();
    for (int64_t i = 1; i < dims; ++i)
        if (t.size(i) != like.size(i)) throw NotHere();
    return static_cast<float*>(t.data_ptr());
}
// the caller's workspace, or memory that is free again, in the order of the stream, when the call returns
struct Workspace {
    at::Tensor held;
    void* data;
    size_t bytes;
    Workspace(PyObject* o, size_t need, const at::Tensor& like, int device)
    {
        if (o == Py_None) held = at::empty({ (int64_t)need }, like.options().dtype(at::kByte));
        else {
            held = on_gpu(o, at::kByte, device);
            if (!held.is_contiguous()) throw NotHere();
        }
        data = held.data_ptr();
        bytes = (size_t)held.numel();
    }
};
// body() -> status; anything that it throws leaves the call to Python
template <typename F> PyObject* judged(bool counted, F body)
{
    int rc = -1;
    if (counted) {
        try {
            rc = body();
        } catch (...) {
            PyErr_Clear();
            rc = -1;
        }
    }
    return PyLong_FromLong(rc);
}

// mix(function, x, W, bias, residual, activation, y, z, device, stream)
PyObject* mix(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 10, [&] {
        const auto call = function<Mix>(args[0]);
        const int device = small(args[8]), act = small(args[5]);
        void* stream = stream_of(args[9]);
        const at::Tensor& x = first_operand(args[1], device);
        const at::ScalarType dt = x.scalar_type();
        const int type = type_of(x), K = channels(x.size(0));
        if (!THPVariable_CheckExact(args[2]) || THPVariable_Unpack(args[2]).dim() != 2) throw NotHere();
        const int N = channels(THPVariable_Unpack(args[2]).size(0));
        const void *W = packed(args[2], dt, device, { N, K }), *bias = packed(args[3], dt, device, { N }, true);
        const Field fx = field(args[1], dt, device, K, x), r = field(args[4], dt, device, N, x, false, false, true);
        const Field y = field(args[6], dt, device, N, x), z = field(args[7], dt, device, N, x, false, false, true);
        const long P = positions(x);
        const WithoutLock unlocked;
        return call(type, P, N, K, fx.data, fx.ld, W, bias, r.data, r.ld, act, z.data, z.ld, y.data, y.ld, stream);
    });
}

// mix_8bit(function, xq, xscale, Wq, wscale, bias, residual, activation, y, device, stream)
PyObject* mix_8bit(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 11, [&] {
        const auto call = function<Mix8bit>(args[0]);
        const int device = small(args[9]), act = small(args[7]);
        void* stream = stream_of(args[10]);
        const at::Tensor& x = first_operand(args[1], device);
        if (x.scalar_type() != at::kFloat8_e4m3fn || !THPVariable_CheckExact(args[8]) || !THPVariable_CheckExact(args[3])) throw NotHere();
        const at::Tensor& out = THPVariable_Unpack(args[8]);
        const int type = type_of(out), K = channels(x.size(0)), N = channels(THPVariable_Unpack(args[3]).size(0));
        const bool pairs = type == TURBOFNO_C64;
        const at::ScalarType dt = out.scalar_type();
        if (pairs && (x.dim() < 3 || x.size(x.dim() - 1) != 2)) throw NotHere();
        const void* W = pairs ? packed(args[3], at::kFloat8_e4m3fn, device, { N, K, 2 }) : packed(args[3], at::kFloat8_e4m3fn, device, { N, K });
        const float *xs = static_cast<float*>(per_position(args[2], device, x, pairs)), *ws = static_cast<float*>(packed(args[4], at::kFloat, device, { N }));
        const void* bias = packed(args[5], dt, device, { N }, true);
        const Field r = field(args[6], dt, device, N, x, false, pairs, true), y = field(args[8], dt, device, N, x, false, pairs);
        const long P = positions(x, pairs), ld = spread(x, pairs ? 2 : 1);
        const void* xq = x.data_ptr();
        const WithoutLock unlocked;
        return call(type, P, N, K, xq, ld, xs, W, ws, bias, r.data, r.ld, act, y.data, y.ld, stream);
    });
}

// mix_backward(input_grad, weight_grad, workspace_bytes, gy, x, W, z, activation, gz, gx, gW, gbias, workspace, device, stream); gz is gy where there is no activation
PyObject* mix_backward(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 15, [&] {
        const auto input = function<InputGrad>(args[0]);
        const auto weight = function<WeightGrad>(args[1]);
        const auto bytes = function<WeightGradBytes>(args[2]);
        const int device = small(args[13]), act = small(args[7]);
        void* stream = stream_of(args[14]);
        const at::Tensor& gy = first_operand(args[3], device);
        const at::Tensor& x = first_operand(args[4], device);
        const at::ScalarType dt = gy.scalar_type();
        const int type = type_of(gy), N = channels(gy.size(0)), K = channels(x.size(0));
        const bool slopes = act != TURBOFNO_ACT_NONE;
        const Field g = field(args[3], dt, device, N, gy), fx = field(args[4], dt, device, K, gy);
        const Field z = slopes ? field(args[6], dt, device, N, gy) : Field(), gz = slopes ? field(args[8], dt, device, N, gy) : g, gx = field(args[9], dt, device, K, gy);
        const void* W = packed(args[5], dt, device, { N, K });
        void *gW = packed(args[10], dt, device, { N, K }), *gbias = packed(args[11], dt, device, { N });
        const long P = positions(gy);
        const Workspace ws(args[12], bytes(type, P, N, K), gy, device);
        // neither call sees what the other one reads or writes
        const size_t e = dt == at::kComplexFloat ? 8 : dt == at::kFloat ? 4 : 2;
        const tfno::Place at_x = tfno::place(fx.data, K, fx.ld, e, P), at_gx = tfno::place(gx.data, K, gx.ld, e, P);
        if (overlap(at_gx, at_x) || (slopes && overlap(tfno::place(gz.data, N, gz.ld, e, P), at_x)) || overlap(tfno::packed(gW, (long)(e * N * K)), at_gx) ||
            overlap(tfno::packed(gbias, (long)(e * N)), at_gx) || overlap(tfno::packed(ws.data, (long)ws.bytes), at_gx))
            throw NotHere();
        const WithoutLock unlocked;
        const int rc = input(type, P, N, K, g.data, g.ld, z.data, z.ld, W, act, slopes ? gz.data : nullptr, gz.ld, gx.data, gx.ld, stream);
        return rc ? rc : weight(type, P, N, K, gz.data, gz.ld, fx.data, fx.ld, gW, gbias, ws.data, ws.bytes, stream);
    });
}

// rms_norm(function, eight bits, x, gain, residual, eps, s, y or q, rstd or scale, device, stream)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 11, [&] {
        const auto call = function<Norm>(args[0]);
        const int eight = small(args[1]), device = small(args[9]);
        void* stream = stream_of(args[10]);
        const at::Tensor& x = first_operand(args[2], device);
        const at::ScalarType dt = x.scalar_type();
        const int type = type_of(x), K = channels(x.size(0));
        const float* gain = static_cast<float*>(packed(args[3], at::kFloat, device, { K }));
        const float eps = real_value(args[5]);
        const Field fx = field(args[2], dt, device, K, x), r = field(args[4], dt, device, K, x, false, false, true), s = field(args[6], dt, device, K, x, false, false, true);
        const Field y = eight ? field(args[7], at::kFloat8_e4m3fn, device, K, x, type == TURBOFNO_C64) : field(args[7], dt, device, K, x);
        float* rstd = static_cast<float*>(per_position(args[8], device, x));
        const long P = positions(x);
        const WithoutLock unlocked;
        return call(type, P, K, fx.data, fx.ld, r.data, r.ld, gain, eps, s.data, s.ld, y.data, y.ld, rstd, stream);
    });
}

// rms_norm_backward(function, workspace_bytes, gy, s, gain, rstd, gs, gx, ggain, workspace, device, stream)
PyObject* rms_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 12, [&] {
        const auto call = function<NormGrad>(args[0]);
        const auto bytes = function<NormGradBytes>(args[1]);
        const int device = small(args[10]);
        void* stream = stream_of(args[11]);
        const at::Tensor& gy = first_operand(args[2], device);
        const at::ScalarType dt = gy.scalar_type();
        const int type = type_of(gy), K = channels(gy.size(0));
        const Field g = field(args[2], dt, device, K, gy), s = field(args[3], dt, device, K, gy), gs = field(args[6], dt, device, K, gy, false, false, true);
        const Field gx = field(args[7], dt, device, K, gy);
        const float* gain = static_cast<float*>(packed(args[4], at::kFloat, device, { K }));
        const float* rstd = static_cast<float*>(per_position(args[5], device, gy));
        float* ggain = static_cast<float*>(packed(args[8], at::kFloat, device, { K }));
        const long P = positions(gy);
        const Workspace ws(args[9], bytes(type, P, K), gy, device);
        const WithoutLock unlocked;
        return call(type, P, K, g.data, g.ld, s.data, s.ld, gain, rstd, gs.data, gs.ld, gx.data, gx.ld, ggain, ws.data, ws.bytes, stream);
    });
}

// dropout(function, x, residual, drop, rng, y, device, stream)
PyObject* dropout(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 8, [&] {
        const auto call = function<Dropout>(args[0]);
        const int device = small(args[6]);
        void* stream = stream_of(args[7]);
        const at::Tensor& x = first_operand(args[1], device);
        const at::ScalarType dt = x.scalar_type();
        const int type = type_of(x), K = channels(x.size(0));
        const Field fx = field(args[1], dt, device, K, x), r = field(args[2], dt, device, K, x, false, false, true), y = field(args[5], dt, device, K, x);
        const double drop = double_value(args[3]);
        const void* rng = seed_and_offset(args[4], device);
        const long P = positions(x);
        const WithoutLock unlocked;
        return call(type, P, K, fx.data, fx.ld, r.data, r.ld, drop, rng, y.data, y.ld, stream);
    });
}

// layer_norm(function, x, gain, bias, residual, eps, drop, rng, s, y, mean, rstd, device, stream)
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 14, [&] {
        const auto call = function<LayerNorm>(args[0]);
        const int device = small(args[12]);
        void* stream = stream_of(args[13]);
        const at::Tensor& x = first_operand(args[1], device);
        const at::ScalarType dt = x.scalar_type();
        const int type = type_of(x), K = channels(x.size(0));
        const float* gain = static_cast<float*>(packed(args[2], at::kFloat, device, { K }));
        const void* bias = packed(args[3], wide(dt), device, { K }, true);
        const float eps = real_value(args[5]);
        const double drop = double_value(args[6]);
        const void* rng = seed_and_offset(args[7], device);
        const Field fx = field(args[1], dt, device, K, x), r = field(args[4], dt, device, K, x, false, false, true), s = field(args[8], dt, device, K, x, false, false, true);
        const Field y = field(args[9], dt, device, K, x);
        void* mean = at_positions(args[10], wide(dt), device, x);
        float* rstd = static_cast<float*>(at_positions(args[11], at::kFloat, device, x));
        const long P = positions(x);
        const WithoutLock unlocked;
        return call(type, P, K, fx.data, fx.ld, r.data, r.ld, gain, bias, eps, drop, rng, s.data, s.ld, y.data, y.ld, mean, rstd, stream);
    });
}

// layer_norm_8bit(function, x, gain, bias, residual, eps, s, q, scale, device, stream)
PyObject* layer_norm_8bit(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 11, [&] {
        const auto call = function<LayerNorm8bit>(args[0]);
        const int device = small(args[9]);
        void* stream = stream_of(args[10]);
        const at::Tensor& x = first_operand(args[1], device);
        const at::ScalarType dt = x.scalar_type();
        const int type = type_of(x), K = channels(x.size(0));
        const float* gain = static_cast<float*>(packed(args[2], at::kFloat, device, { K }));
        const void* bias = packed(args[3], wide(dt), device, { K }, true);
        const float eps = real_value(args[5]);
        const Field fx = field(args[1], dt, device, K, x), r = field(args[4], dt, device, K, x, false, false, true), s = field(args[6], dt, device, K, x, false, false, true);
        const Field q = field(args[7], at::kFloat8_e4m3fn, device, K, x, type == TURBOFNO_C64);
        float* scale = block_scales(args[8], device, K, x);
        const long P = positions(x);
        const WithoutLock unlocked;
        return call(type, P, K, fx.data, fx.ld, r.data, r.ld, gain, bias, eps, s.data, s.ld, q.data, q.ld, scale, stream);
    });
}

// layer_norm_backward(function, workspace_bytes, gy, s, gain, mean, rstd, gs, drop, rng, gx, gr, ggain, gbias, workspace, device, stream); gr: None without dropout
PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 17, [&] {
        const auto call = function<LayerNormGrad>(args[0]);
        const auto bytes = function<LayerNormGradBytes>(args[1]);
        const int device = small(args[15]);
        void* stream = stream_of(args[16]);
        const at::Tensor& gy = first_operand(args[2], device);
        const at::ScalarType dt = gy.scalar_type();
        const int type = type_of(gy), K = channels(gy.size(0));
        const Field g = field(args[2], dt, device, K, gy), s = field(args[3], dt, device, K, gy), gs = field(args[7], dt, device, K, gy, false, false, true);
        const float* gain = static_cast<float*>(packed(args[4], at::kFloat, device, { K }));
        const void* mean = at_positions(args[5], wide(dt), device, gy);
        const float* rstd = static_cast<float*>(at_positions(args[6], at::kFloat, device, gy));
        const double drop = double_value(args[8]);
        const void* rng = seed_and_offset(args[9], device);
        const Field gx = field(args[10], dt, device, K, gy), gr = field(args[11], dt, device, K, gy, false, false, true);
        float* ggain = static_cast<float*>(packed(args[12], at::kFloat, device, { K }));
        void* gbias = packed(args[13], wide(dt), device, { K });
        const long P = positions(gy);
        const Workspace ws(args[14], bytes(type, P, K), gy, device);
        const WithoutLock unlocked;
        return call(type, P, K, g.data, g.ld, s.data, s.ld, gain, mean, rstd, gs.data, gs.ld, drop, rng, gr.data, gr.ld, gx.data, gx.ld, ggain, gbias, ws.data, ws.bytes,
                    stream);
    });
}

// quantise_8bit(function, x, q, scale, device, stream)
PyObject* quantise_8bit(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 6, [&] {
        const auto call = function<Quantise>(args[0]);
        const int device = small(args[4]);
        void* stream = stream_of(args[5]);
        const at::Tensor& x = first_operand(args[1], device);
        const int type = type_of(x), K = channels(x.size(0));
        const Field fx = field(args[1], x.scalar_type(), device, K, x), q = field(args[2], at::kFloat8_e4m3fn, device, K, x, type == TURBOFNO_C64);
        float* scale = block_scales(args[3], device, K, x);
        const long P = positions(x);
        const WithoutLock unlocked;
        return call(type, P, K, fx.data, fx.ld, q.data, q.ld, scale, stream);
    });
}

// mix_8bit_blocks(function, xq, xscale, Wq, wscale, bias, residual, activation, y, device, stream)
PyObject* mix_8bit_blocks(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 11, [&] {
        const auto call = function<Mix8bitBlocks>(args[0]);
        const int device = small(args[9]), act = small(args[7]);
        void* stream = stream_of(args[10]);
        const at::Tensor& x = first_operand(args[1], device);
        if (x.scalar_type() != at::kFloat8_e4m3fn || !THPVariable_CheckExact(args[8]) || !THPVariable_CheckExact(args[3])) throw NotHere();
        const at::Tensor& out = THPVariable_Unpack(args[8]);
        if (THPVariable_Unpack(args[3]).dim() < 2) throw NotHere();
        const int type = type_of(out), K = channels(x.size(0)), N = channels(THPVariable_Unpack(args[3]).size(0));
        const bool pairs = type == TURBOFNO_C64;
        const at::ScalarType dt = out.scalar_type();
        if (pairs && (x.dim() < 3 || x.size(x.dim() - 1) != 2)) throw NotHere();
        const void* W = pairs ? packed(args[3], at::kFloat8_e4m3fn, device, { N, K, 2 }) : packed(args[3], at::kFloat8_e4m3fn, device, { N, K });
        const float *xs = block_scales(args[2], device, K, x, pairs), *ws = static_cast<float*>(packed(args[4], at::kFloat, device, { (N + 127) / 128, (K + 127) / 128 }));
        const void* bias = packed(args[5], dt, device, { N }, true);
        const Field r = field(args[6], dt, device, N, x, false, pairs, true), y = field(args[8], dt, device, N, x, false, pairs);
        const long P = positions(x, pairs), ld = spread(x, pairs ? 2 : 1);
        const void* xq = x.data_ptr();
        const WithoutLock unlocked;
        return call(type, P, N, K, xq, ld, xs, W, ws, bias, r.data, r.ld, act, y.data, y.ld, stream);
    });
}

// clip_grad_norm(function, workspace_bytes, list of gradients, list of results, max_norm, norm, workspace, device, stream)
PyObject* clip_grad_norm(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    return judged(count == 9, [&] {
        const auto call = function<Clip>(args[0]);
        const auto bytes = function<ClipBytes>(args[1]);
        const int device = small(args[7]);
        void* stream = stream_of(args[8]);
        if (!PyList_CheckExact(args[2]) || !PyList_CheckExact(args[3]) || PyList_GET_SIZE(args[2]) != PyList_GET_SIZE(args[3]) || PyList_GET_SIZE(args[2]) > INT_MAX)
            throw NotHere();
        const int n = (int)PyList_GET_SIZE(args[2]);
        const float max_norm = real_value(args[4]);
        std::vector<const void*> grads(n);
        std::vector<void*> out(n);
        std::vector<long> sizes(n);
        std::vector<int> types(n);
        for (int i = 0; i < n; ++i) {
            PyObject *go = PyList_GET_ITEM(args[2], i), *oo = PyList_GET_ITEM(args[3], i);
            if (!THPVariable_CheckExact(go)) throw NotHere();
            const at::Tensor& g = on_gpu(go, THPVariable_Unpack(go).scalar_type(), device);
            const at::Tensor& o = go == oo ? g : on_gpu(oo, g.scalar_type(), device);
            if (!g.is_contiguous() || !o.is_contiguous() || o.sizes() != g.sizes()) throw NotHere();
            types[i] = type_of(g);
            sizes[i] = g.numel();
            grads[i] = g.data_ptr();
            out[i] = o.data_ptr();
        }
        float* norm = static_cast<float*>(packed(args[5], at::kFloat, device, {}));
        const Workspace ws(args[6], bytes(n), THPVariable_Unpack(args[5]), device);
        const WithoutLock unlocked;
        return call(n, grads.data(), out.data(), sizes.data(), types.data(), max_norm, norm, ws.data, ws.bytes, stream);
    });
}

PyMethodDef methods[] = {
    { "operands", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(operands)), METH_FASTCALL, "addresses of complex64 GPU tensors of given sizes, or None" },
    { "layer_1d", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_1d)), METH_FASTCALL, "turbofno_layer_1d on checked tensors, or -1" },
    { "layer_2d", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_2d)), METH_FASTCALL, "turbofno_layer_2d on checked tensors, or -1" },
#define TFNO_METHOD(name, text) { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, text }
    TFNO_METHOD(mix, "turbofno_mix on checked tensors, or -1"),
    TFNO_METHOD(mix_8bit, "turbofno_mix_8bit on checked tensors, or -1"),
    TFNO_METHOD(mix_backward, "turbofno_mix_input_grad and turbofno_mix_weight_grad on checked tensors, or -1"),
    TFNO_METHOD(rms_norm, "turbofno_rms_norm or turbofno_rms_norm_8bit on checked tensors, or -1"),
    TFNO_METHOD(rms_norm_backward, "turbofno_rms_norm_backward on checked tensors, or -1"),
    TFNO_METHOD(dropout, "turbofno_dropout on checked tensors, or -1"),
    TFNO_METHOD(layer_norm, "turbofno_layer_norm on checked tensors, or -1"),
    TFNO_METHOD(layer_norm_8bit, "turbofno_layer_norm_8bit on checked tensors, or -1"),
    TFNO_METHOD(layer_norm_backward, "turbofno_layer_norm_backward on checked tensors, or -1"),
    TFNO_METHOD(quantise_8bit, "turbofno_quantise_8bit on checked tensors, or -1"),
    TFNO_METHOD(mix_8bit_blocks, "turbofno_mix_8bit_blocks on checked tensors, or -1"),
    TFNO_METHOD(clip_grad_norm, "turbofno_clip_grad_norm on lists of checked tensors, or -1"),
    { nullptr, nullptr, 0, nullptr },
};
PyModuleDef module = { PyModuleDef_HEAD_INIT, "_operands", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr };

}  // namespace

// BUILT_FOR: torch and Python of the headers, "torch <version>, <SOABI>"; the binding leaves the module alone under any other
PyMODINIT_FUNC PyInit__operands(void)
{
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", BUILT_FOR) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
