// Host path of the linears, of the microscaled 4-bit tier and of expert routing:
// one native call per forward for the calls a model makes (contiguous GPU
// activations, operands as the layers keep them, no trace).  It checks the operands, allocates the output and the intermediates and calls the
// library; anything else returns None and takes the Python path, which handles
// every form and raises the errors.
//
// The intermediates come from torch's caching allocator on the current stream
// and go back to it when the call returns, which orders their reuse on that
// stream; nothing is kept between calls.  Shapes whose GEMM splits k over
// workgroups need a workspace with cleared counters and are left to Python,
// which keeps one per stream.
//
// Measured on MI355X (M = 1, 256 x 256, back to back): 17.3 us per W4A4
// call through Python and ctypes, 7.1 here; 21.9 and 9.5 with a LoRA; W8A8 27.2
// (16.0 as one library call) and 6.8.

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/ATen.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>

#include "../../include/convrot_mi355x.h"

namespace {

// f32 0, bf16 1, f16 2 (the library's dtype codes), -1: none of them
int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

constexpr int kEpiF16 = 5;

// A plain strided GPU tensor on `dev`, contiguous, its data 16-byte aligned and there (a functional tensor's is not).
bool plain(const at::Tensor& t, c10::Device dev) {
    return t.defined() && t.layout() == at::kStrided && t.device() == dev && !t.is_neg() && t.has_storage() &&
           t.is_contiguous() && (t.const_data_ptr() != nullptr || t.numel() == 0) &&
           reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}

// None, or a tensor of exactly torch.Tensor / Parameter type; false for other objects
bool optional_tensor(PyObject* o, at::Tensor* t) {
    if (o == Py_None) return true;
    if (!THPVariable_CheckExact(o)) return false;
    *t = THPVariable_Unpack(o);
    return true;
}

struct Linear {
    at::Tensor x, w, scales, bias;
    int64_t M, N, K;
    int xdt, bdt, odt, epi;
};

// The operands common to the linears; K and N from the caller.  False: not a call for this path.
bool common(Linear& l, PyObject* ox, PyObject* os, PyObject* ob) {
    if (!THPVariable_CheckExact(ox) || !THPVariable_CheckExact(os)) return false;
    if (c10::impl::TorchDispatchModeTLS::any_modes_set()) return false;   // modes see the Python path's operations
    l.x = THPVariable_Unpack(ox);
    l.scales = THPVariable_Unpack(os);
    if (!l.x.is_cuda() || l.x.dim() < 1 || !optional_tensor(ob, &l.bias)) return false;
    const c10::Device dev = l.x.device();
    if (dev.index() != c10::hip::current_device() || !plain(l.x, dev) || !plain(l.scales, dev)) return false;
    l.xdt = dtype_code(l.x);
    l.K = l.x.size(-1);
    if (l.xdt < 0 || l.K <= 0 || l.x.numel() == 0 || l.scales.scalar_type() != at::kFloat) return false;
    const int64_t M = l.x.numel() / l.K;
    if (M > INT32_MAX) return false;
    l.M = M;
    l.bdt = 0;
    if (l.bias.defined()) {
        l.bdt = dtype_code(l.bias);
        if (l.bdt < 0 || !plain(l.bias, dev)) return false;
    }
    return true;
}

at::Tensor empty_out(const Linear& l) {
    std::vector<int64_t> sizes(l.x.sizes().begin(), l.x.sizes().end());
    sizes.back() = l.N;
    return at::empty(sizes, l.x.options().requires_grad(false));
}

int group_of(PyObject* o) {
    if (!PyLong_CheckExact(o)) return -1;
    const long g = PyLong_AsLong(o);
    if (g == -1 && PyErr_Occurred()) { PyErr_Clear(); return -1; }
    return g == 16 || g == 64 || g == 256 ? (int)g : -1;
}

const void* ptr(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

PyObject* finish(int rc, const char* what, at::Tensor out) {
    if (rc != 0) {
        PyErr_Format(PyExc_RuntimeError, "%s failed, hipError=%d", what, rc);
        return nullptr;
    }
    return THPVariable_Wrap(std::move(out));
}

// w4a4(x, qweight, wscales, bias, groupsize, eager, lora, qweight_bf6)
PyObject* w4a4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Linear l;
    if (n != 8 || !common(l, a[0], a[2], a[3]) || !THPVariable_CheckExact(a[1])) Py_RETURN_NONE;
    const c10::Device dev = l.x.device();
    const at::Tensor& qw = THPVariable_Unpack(a[1]);
    const int G = group_of(a[4]);
    if (G < 0 || l.K % G != 0 || qw.dim() != 2 || qw.size(1) * 2 != l.K || qw.size(0) < 1) Py_RETURN_NONE;
    l.N = qw.size(0);
    if (l.N > INT32_MAX || l.scales.numel() != l.N || (l.bias.defined() && l.bias.numel() != l.N)) Py_RETURN_NONE;
    const bool bf6 = l.K % 128 == 0 && l.K <= cr_max_quant_bf6_k();
    if (bf6) {
        if (!THPVariable_CheckExact(a[7])) Py_RETURN_NONE;
        l.w = THPVariable_Unpack(a[7]);
        if (!plain(l.w, dev) || l.w.scalar_type() != at::kByte || l.w.dim() != 2 || l.w.size(1) != l.K / 4 * 3 ||
            l.w.size(0) != (l.N + 255) / 256 * 256)
            Py_RETURN_NONE;
    } else {
        l.w = qw;
        if (l.K % 64 != 0 || l.K > cr_max_quant_k() || !plain(l.w, dev) || l.w.scalar_type() != at::kChar) Py_RETURN_NONE;
    }
    at::Tensor down, up;
    int R = 0;
    if (a[6] != Py_None) {
        if (!PyTuple_CheckExact(a[6]) || PyTuple_GET_SIZE(a[6]) != 2) Py_RETURN_NONE;
        PyObject *od = PyTuple_GET_ITEM(a[6], 0), *ou = PyTuple_GET_ITEM(a[6], 1);
        if (l.xdt == 0 || !THPVariable_CheckExact(od) || !THPVariable_CheckExact(ou)) Py_RETURN_NONE;
        down = THPVariable_Unpack(od);
        up = THPVariable_Unpack(ou);
        if (!plain(down, dev) || !plain(up, dev) || down.scalar_type() != at::kBFloat16 ||
            up.scalar_type() != at::kBFloat16 || down.dim() != 2 || up.dim() != 2 || down.size(1) != l.K ||
            up.size(0) != l.N || up.size(1) != down.size(0) || down.size(0) > 128 || down.size(0) < 32 ||
            down.size(0) % 32 != 0)
            Py_RETURN_NONE;
        R = (int)down.size(0);
    }
    const int M = (int)l.M, N = (int)l.N, K = (int)l.K;
    if (bf6 && cr_convrot_w4a4_linear_bf6_split(M, N, K)) Py_RETURN_NONE;
    const size_t ws_bytes = bf6 ? cr_convrot_w4a4_linear_bf6_min_workspace(M, N, K, R)
                                : cr_convrot_w4a4_linear_packed_workspace(M, N, K, R);
    const int epi = l.xdt == 1 ? (a[5] == Py_True ? 2 : 1) : 0;
    int rc;
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        out = empty_out(l);
        const at::Tensor ws = at::empty({(int64_t)ws_bytes}, l.x.options().dtype(at::kByte).requires_grad(false));
        void* st = c10::hip::getCurrentHIPStream(dev.index()).stream();
        if (bf6 && l.xdt == 2)
            rc = cr_convrot_w4a4_linear_bf6_f16(l.x.const_data_ptr(), l.xdt, l.w.const_data_ptr(), l.scales.const_data_ptr(),
                                                ptr(l.bias), l.bdt, ptr(down), ptr(up), R, 1.0f, out.mutable_data_ptr(), M, N,
                                                K, G, ws.mutable_data_ptr(), ws_bytes, st);
        else if (bf6)
            rc = cr_convrot_w4a4_linear_bf6(l.x.const_data_ptr(), l.xdt, l.w.const_data_ptr(), l.scales.const_data_ptr(),
                                            ptr(l.bias), l.bdt, ptr(down), ptr(up), R, 1.0f, out.mutable_data_ptr(), epi, M,
                                            N, K, G, ws.mutable_data_ptr(), ws_bytes, st);
        else
            rc = cr_convrot_w4a4_linear_packed(l.x.const_data_ptr(), l.xdt, l.w.const_data_ptr(), l.scales.const_data_ptr(),
                                               ptr(l.bias), l.bdt, ptr(down), ptr(up), R, 1.0f, out.mutable_data_ptr(),
                                               l.xdt == 2 ? kEpiF16 : epi, M, N, K, G, ws.mutable_data_ptr(), ws_bytes, st);
    }
    return finish(rc, "the W4A4 linear", std::move(out));
    END_HANDLE_TH_ERRORS
}

// w8a8(x, qweight, wscales, bias, groupsize, qweight_i8t)
PyObject* w8a8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Linear l;
    if (n != 6 || !common(l, a[0], a[2], a[3]) || !THPVariable_CheckExact(a[1]) || !THPVariable_CheckExact(a[5]))
        Py_RETURN_NONE;
    const c10::Device dev = l.x.device();
    const at::Tensor& qw = THPVariable_Unpack(a[1]);
    l.w = THPVariable_Unpack(a[5]);
    const int G = group_of(a[4]);
    if (G < 0 || l.K % G != 0 || l.K % 64 != 0 || l.K > cr_max_quant_bf6_k() || qw.dim() != 2 || qw.size(1) != l.K ||
        qw.size(0) < 1)
        Py_RETURN_NONE;
    l.N = qw.size(0);
    if (l.N > INT32_MAX || l.scales.numel() != l.N || (l.bias.defined() && l.bias.numel() != l.N) || !plain(l.w, dev) ||
        l.w.scalar_type() != at::kChar || l.w.dim() != 2 || l.w.size(1) != l.K || l.w.size(0) != (l.N + 255) / 256 * 256)
        Py_RETURN_NONE;
    const int M = (int)l.M, N = (int)l.N, K = (int)l.K;
    if (cr_convrot_w8a8_linear_i8t_split(M, N, K)) Py_RETURN_NONE;
    const size_t ws_bytes = cr_convrot_w8a8_linear_i8t_workspace(M, N, K);
    int rc;
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        out = empty_out(l);
        const at::Tensor ws = at::empty({(int64_t)ws_bytes}, l.x.options().dtype(at::kByte).requires_grad(false));
        void* st = c10::hip::getCurrentHIPStream(dev.index()).stream();
        rc = cr_convrot_w8a8_linear_i8t(l.x.const_data_ptr(), l.xdt, l.w.const_data_ptr(),
                                        l.scales.const_data_ptr(), ptr(l.bias), l.bdt, out.mutable_data_ptr(),
                                        l.xdt == 2 ? kEpiF16 : l.xdt, M, N, K, G, ws.mutable_data_ptr(), ws_bytes, st);
    }
    return finish(rc, "the W8A8 linear", std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// Microscaled 4-bit tier (_int4/mxfp4.py) and expert routing (_int4/experts.py):
// the same checks' good side; whatever fails one takes the Python path, which
// says why.  Measured on MI355X (back to back): 13.5 us a linear of 1 x 5120 ->
// 13824 through Python and ctypes, 9.4 here, what its kernel takes; 12.1 and 5.3 of
// 1 x 4096 -> 4096.
// ---------------------------------------------------------------------------

// A tensor for these paths: exactly torch.Tensor or Parameter, plain, on the current device, without a forward gradient.
bool operand(PyObject* o, at::Tensor* t, c10::Device* dev, bool first = false) {
    if (!THPVariable_CheckExact(o)) return false;
    *t = THPVariable_Unpack(o);
    if (!t->is_cuda() || t->_fw_grad(0).defined()) return false;
    if (first) {
        if (c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing()) return false;
        *dev = t->device();
        if (dev->index() != c10::hip::current_device()) return false;
    }
    return plain(*t, *dev);
}

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }

// None -> 0, 16, 64 or 256; -1: not one of them, or K is not whole groups and blocks or past what the library takes
int mx_group(PyObject* o, int64_t K) {
    if (K <= 0 || K % 32 != 0 || K > (1 << 24)) return -1;
    if (o == Py_None) return 0;
    const int G = group_of(o);
    return G > 0 && K % G == 0 ? G : -1;
}

at::Tensor like(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
    return at::empty(sizes, t.options().dtype(type).requires_grad(false));
}

void* stream_of(c10::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

// mx_quantize(x, groupsize) -> (codes, scales)
PyObject* mx_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor x;
    c10::Device dev(c10::kCPU);
    if (n != 2 || !operand(a[0], &x, &dev, true) || x.dim() < 1 || wants_grad(x)) Py_RETURN_NONE;
    const int dt = dtype_code(x);
    const int64_t K = x.size(-1);
    const int G = mx_group(a[1], K);
    if (dt < 0 || G < 0 || x.numel() == 0 || x.numel() / K > INT32_MAX) Py_RETURN_NONE;
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = K / 2;
    at::Tensor codes = like(x, sizes, at::kByte);
    sizes.back() = K / 32;
    at::Tensor scales = like(x, sizes, at::kByte);
    const int rc = cr_mxfp4_quant(x.const_data_ptr(), dt, codes.mutable_data_ptr(), scales.mutable_data_ptr(),
                                  (int)(x.numel() / K), (int)K, G, stream_of(dev));
    if (rc != 0) return finish(rc, "cr_mxfp4_quant", codes);
    return PyTuple_Pack(2, pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(codes))).ptr(),
                        pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(scales))).ptr());
    END_HANDLE_TH_ERRORS
}

// mx_dequantize(codes, scales, groupsize, dtype code)
PyObject* mx_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor codes, scales;
    c10::Device dev(c10::kCPU);
    if (n != 4 || !operand(a[0], &codes, &dev, true) || !operand(a[1], &scales, &dev) || codes.dim() < 1) Py_RETURN_NONE;
    const int64_t K = codes.size(-1) * 2;
    const int G = mx_group(a[2], K);
    const long dt = PyLong_AsLong(a[3]);
    if (G < 0 || dt < 0 || dt > 2 || codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte ||
        codes.numel() == 0 || codes.numel() * 2 / K > INT32_MAX || scales.dim() != codes.dim() || scales.size(-1) != K / 32 ||
        scales.sizes().slice(0, scales.dim() - 1) != codes.sizes().slice(0, codes.dim() - 1))
        Py_RETURN_NONE;
    std::vector<int64_t> sizes(codes.sizes().begin(), codes.sizes().end());
    sizes.back() = K;
    at::Tensor out = like(codes, sizes, dt == 0 ? at::kFloat : dt == 1 ? at::kBFloat16 : at::kHalf);
    const int rc = cr_mxfp4_dequant(codes.const_data_ptr(), scales.const_data_ptr(), out.mutable_data_ptr(), (int)dt,
                                    (int)(out.numel() / K), (int)K, G, stream_of(dev));
    return finish(rc, "cr_mxfp4_dequant", std::move(out));
    END_HANDLE_TH_ERRORS
}

// The weight of a product: codes [.., N, K/2], scales [.., N, K/32], bias None or [.., N]
bool mx_weight(PyObject* ow, PyObject* os, PyObject* ob, c10::Device dev, int64_t dim, int64_t K, at::Tensor* w, at::Tensor* s,
               at::Tensor* b, int* bdt) {
    c10::Device d = dev;
    if (!operand(ow, w, &d) || !operand(os, s, &d) || w->dim() != dim || w->size(-1) * 2 != K || w->numel() == 0 ||
        w->scalar_type() != at::kByte || s->scalar_type() != at::kByte || s->dim() != dim || s->size(-1) != K / 32 ||
        s->sizes().slice(0, dim - 1) != w->sizes().slice(0, dim - 1) || w->size(-2) > 0x7fffff00)
        return false;
    *bdt = 0;
    if (ob == Py_None) return true;
    if (!operand(ob, b, &d) || b->sizes() != w->sizes().slice(0, dim - 1) || wants_grad(*b)) return false;
    *bdt = dtype_code(*b);
    return *bdt >= 0;
}

// mx_linear(x, qweight, wscales, bias, groupsize)
PyObject* mx_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor x, w, s, b;
    c10::Device dev(c10::kCPU);
    int bdt;
    if (n != 5 || !operand(a[0], &x, &dev, true) || x.dim() < 1 || wants_grad(x)) Py_RETURN_NONE;
    const int dt = dtype_code(x);
    const int64_t K = x.size(-1);
    const int G = mx_group(a[4], K);
    if (dt < 0 || G < 0 || x.numel() == 0 || x.numel() / K > INT32_MAX || !mx_weight(a[1], a[2], a[3], dev, 2, K, &w, &s, &b, &bdt))
        Py_RETURN_NONE;
    const int M = (int)(x.numel() / K), N = (int)w.size(0);
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = N;
    at::Tensor out = like(x, sizes, x.scalar_type());
    const size_t bytes = cr_mxfp4_linear_workspace(M, N, (int)K, 1);
    const at::Tensor ws = like(x, {(int64_t)bytes}, at::kByte);
    const int rc = cr_mxfp4_linear(x.const_data_ptr(), dt, w.const_data_ptr(), s.const_data_ptr(), ptr(b), bdt,
                                   out.mutable_data_ptr(), M, N, (int)K, G, ws.mutable_data_ptr(), bytes, stream_of(dev));
    return finish(rc, "cr_mxfp4_linear", std::move(out));
    END_HANDLE_TH_ERRORS
}

// The tensors of a plan: order [T k], position [T, k], offsets [E + 1], int32
struct Plan {
    at::Tensor order, position, offsets;
    int T, k, E;
    bool take(PyObject* oo, PyObject* op, PyObject* of, c10::Device dev) {
        if (!operand(oo, &order, &dev) || !operand(op, &position, &dev) || !operand(of, &offsets, &dev) || order.dim() != 1 ||
            position.dim() != 2 || offsets.dim() != 1 || order.scalar_type() != at::kInt || position.scalar_type() != at::kInt ||
            offsets.scalar_type() != at::kInt || order.numel() == 0 || order.numel() != position.numel() ||
            order.numel() > INT32_MAX || offsets.numel() < 2 || offsets.numel() > 1 + cr_max_experts())
            return false;
        T = (int)position.size(0);
        k = (int)position.size(1);
        E = (int)offsets.numel() - 1;
        return true;
    }
};

// mx_expert_linear(x, qweight, wscales, order, position, offsets, bias, groupsize, sorted)
PyObject* mx_expert_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor x, w, s, b;
    Plan p;
    c10::Device dev(c10::kCPU);
    int bdt;
    if (n != 9 || !operand(a[0], &x, &dev, true) || x.dim() != 2 || wants_grad(x) || !p.take(a[3], a[4], a[5], dev)) Py_RETURN_NONE;
    const int dt = dtype_code(x);
    const int64_t K = x.size(1);
    const int G = mx_group(a[7], K);
    const bool sorted = a[8] == Py_True;
    if (dt < 0 || G < 0 || !mx_weight(a[1], a[2], a[6], dev, 3, K, &w, &s, &b, &bdt) || w.size(0) != p.E ||
        x.size(0) != (sorted ? (int64_t)p.T * p.k : p.T))
        Py_RETURN_NONE;
    const int R = p.T * p.k, N = (int)w.size(1);
    at::Tensor out = like(x, {R, N}, x.scalar_type());
    const size_t bytes = cr_mxfp4_linear_workspace((int)x.size(0), N, (int)K, p.E);
    const at::Tensor ws = like(x, {(int64_t)bytes}, at::kByte);
    const int rc = cr_mxfp4_expert_linear(x.const_data_ptr(), dt, sorted ? nullptr : (const int*)p.order.const_data_ptr(), p.k,
                                          (const int*)p.offsets.const_data_ptr(), p.E, w.const_data_ptr(), s.const_data_ptr(), ptr(b),
                                          bdt, out.mutable_data_ptr(), R, N, (int)K, G, ws.mutable_data_ptr(), bytes,
                                          stream_of(dev));
    return finish(rc, "cr_mxfp4_expert_linear", std::move(out));
    END_HANDLE_TH_ERRORS
}

// expert_sort(ids, experts) -> (order, position, offsets)
PyObject* expert_sort(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor ids;
    c10::Device dev(c10::kCPU);
    if (n != 2 || !operand(a[0], &ids, &dev, true) || ids.dim() != 2 || ids.numel() == 0 || ids.numel() > INT32_MAX ||
        (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) || !PyLong_CheckExact(a[1]))
        Py_RETURN_NONE;
    const long E = PyLong_AsLong(a[1]);
    if (E == -1 && PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (E < 1 || E > cr_max_experts()) Py_RETURN_NONE;
    const int R = (int)ids.numel();
    at::Tensor order = like(ids, {R}, at::kInt), position = like(ids, ids.sizes(), at::kInt), offsets = like(ids, {E + 1}, at::kInt);
    const size_t bytes = cr_expert_sort_workspace(R, (int)E);
    const at::Tensor ws = like(ids, {(int64_t)bytes}, at::kByte);
    const int rc = cr_expert_sort(ids.const_data_ptr(), (int)ids.element_size(), (int*)order.mutable_data_ptr(),
                                  (int*)position.mutable_data_ptr(), (int*)offsets.mutable_data_ptr(), R, (int)E,
                                  ws.mutable_data_ptr(), bytes, stream_of(dev));
    if (rc != 0) return finish(rc, "cr_expert_sort", order);
    return PyTuple_Pack(3, pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(order))).ptr(),
                        pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(position))).ptr(),
                        pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::move(offsets))).ptr());
    END_HANDLE_TH_ERRORS
}

at::Tensor gather_rows(const at::Tensor& x, const at::Tensor& position, const at::Tensor& offsets) {
    const int T = (int)position.size(0), k = (int)position.size(1), D = (int)x.size(1);
    at::Tensor rows = like(x, {(int64_t)T * k, D}, x.scalar_type());
    const int rc = cr_expert_gather(x.const_data_ptr(), dtype_code(x), (const int*)position.const_data_ptr(),
                                    (const int*)offsets.const_data_ptr(), rows.mutable_data_ptr(), T, k, (int)offsets.numel() - 1, D,
                                    stream_of(x.device()));
    TORCH_CHECK(rc == 0, "cr_expert_gather failed, hipError=", rc);
    return rows;
}

// weights undefined: 1
at::Tensor combine_rows(const at::Tensor& rows, const at::Tensor& weights, const at::Tensor& position) {
    const int T = (int)position.size(0), k = (int)position.size(1), D = (int)rows.size(1);
    at::Tensor out = like(rows, {T, D}, rows.scalar_type());
    const int rc = cr_expert_combine(rows.const_data_ptr(), dtype_code(rows), (const float*)ptr(weights),
                                     (const int*)position.const_data_ptr(), out.mutable_data_ptr(), T, k, D, stream_of(rows.device()));
    TORCH_CHECK(rc == 0, "cr_expert_combine failed, hipError=", rc);
    return out;
}

// A gradient's own form: its values as they are read, contiguous, aligned
at::Tensor settled(const at::Tensor& t) {
    at::Tensor c = t.resolve_neg().contiguous();
    return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 != 0 ? c.clone() : c;
}

// A saved tensor as the kernels take it: hooks on saved tensors may hand back another one than was saved.
at::Tensor restored(const at::Tensor& t, const char* what, at::ScalarType type, at::IntArrayRef sizes, c10::Device dev) {
    TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.device() == dev && t.scalar_type() == type && t.sizes() == sizes,
                "the saved ", what, " came back in another form: ", type, " ", sizes, " on ", dev, " expected, got ",
                t.toString(), " ", t.sizes(), " on ", t.device());
    return settled(t.detach());
}

// The saved positions [T, k] of T tokens' slots, or of any number of tokens (T < 0)
at::Tensor restored_position(const at::Tensor& t, int64_t T, c10::Device dev) {
    TORCH_CHECK(t.dim() == 2 && t.size(1) >= 1 && t.numel() <= INT32_MAX && (T < 0 || t.size(0) == T),
                "the saved positions came back in another form: ", t.sizes());
    return restored(t, "positions", at::kInt, t.sizes(), dev);
}

// Gradients that cannot be differentiated again: where a graph of them is built, using it raises.
torch::autograd::variable_list once(torch::autograd::variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    torch::autograd::variable_list in;
    std::vector<size_t> where;
    for (size_t i = 0; i < grads.size(); ++i)
        if (grads[i].defined()) {
            in.push_back(grads[i].detach().requires_grad_(true));
            where.push_back(i);
        }
    auto error = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)in.size());
    const torch::autograd::variable_list out = (*error)(std::move(in));
    for (size_t i = 0; i < where.size(); ++i) grads[where[i]] = out[i];
    return grads;
}

struct GatherRows : torch::autograd::Function<GatherRows> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& position,
                              const at::Tensor& offsets) {
        ctx->save_for_backward({position});
        return gather_rows(x, position, offsets);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        at::Tensor d_x;
        {
            at::NoGradGuard no_grad;
            const at::Tensor position = restored_position(ctx->get_saved_variables()[0], -1, g[0].device());
            TORCH_CHECK(position.numel() == g[0].size(0), "the saved positions came back in another form: ", position.sizes());
            d_x = combine_rows(settled(g[0]), at::Tensor(), position);
        }
        return once({d_x, at::Tensor(), at::Tensor()});
    }
};

struct CombineRows : torch::autograd::Function<CombineRows> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& rows, const at::Tensor& weights,
                              const at::Tensor& position, const at::Tensor& offsets) {
        ctx->save_for_backward({rows, weights, position, offsets});
        ctx->saved_data["offsets"] = offsets.numel();
        return combine_rows(rows, weights, position);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        at::Tensor d_rows, d_w;
        {
            at::NoGradGuard no_grad;
            const auto saved = ctx->get_saved_variables();
            const at::Tensor d_out = settled(g[0]);                      // [T, D], which autograd has checked
            const c10::Device dev = d_out.device();
            const at::Tensor position = restored_position(saved[2], d_out.size(0), dev);
            const at::Tensor rows = restored(saved[0], "rows", d_out.scalar_type(), {position.numel(), d_out.size(1)}, dev);
            const at::Tensor w = restored(saved[1], "weights", at::kFloat, position.sizes(), dev);
            const at::Tensor offsets = restored(saved[3], "offsets", at::kInt, {ctx->saved_data["offsets"].toInt()}, dev);
            if (ctx->needs_input_grad(0)) d_rows = like(rows, rows.sizes(), rows.scalar_type());
            if (ctx->needs_input_grad(1)) d_w = like(w, w.sizes(), at::kFloat);
            const int rc = cr_expert_combine_grad(
                    rows.const_data_ptr(), dtype_code(rows), (const float*)w.const_data_ptr(), (const int*)position.const_data_ptr(),
                    (const int*)offsets.const_data_ptr(), d_out.const_data_ptr(), d_rows.defined() ? d_rows.mutable_data_ptr() : nullptr,
                    d_w.defined() ? (float*)d_w.mutable_data_ptr() : nullptr, (int)position.size(0), (int)position.size(1),
                    (int)offsets.numel() - 1, (int)rows.size(1), stream_of(rows.device()));
            TORCH_CHECK(rc == 0, "cr_expert_combine_grad failed, hipError=", rc);
        }
        return once({d_rows, d_w, at::Tensor(), at::Tensor()});
    }
};

// expert_gather(x, order, position, offsets)
PyObject* expert_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor x;
    Plan p;
    c10::Device dev(c10::kCPU);
    if (n != 4 || !operand(a[0], &x, &dev, true) || x.dim() != 2 || dtype_code(x) < 0 || !p.take(a[1], a[2], a[3], dev) ||
        x.size(0) != p.T || x.size(1) < 1 || x.size(1) > INT32_MAX)
        Py_RETURN_NONE;
    return THPVariable_Wrap(wants_grad(x) ? GatherRows::apply(x, p.position, p.offsets) : gather_rows(x, p.position, p.offsets));
    END_HANDLE_TH_ERRORS
}

// expert_combine(rows, weights, order, position, offsets): weights f32
PyObject* expert_combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor rows, w;
    Plan p;
    c10::Device dev(c10::kCPU);
    if (n != 5 || !operand(a[0], &rows, &dev, true) || rows.dim() != 2 || dtype_code(rows) < 0 || !operand(a[1], &w, &dev) ||
        w.scalar_type() != at::kFloat || !p.take(a[2], a[3], a[4], dev) || rows.size(0) != (int64_t)p.T * p.k ||
        rows.size(1) < 1 || rows.size(1) > INT32_MAX || w.sizes() != p.position.sizes())
        Py_RETURN_NONE;
    return THPVariable_Wrap(wants_grad(rows) || wants_grad(w) ? CombineRows::apply(rows, w, p.position, p.offsets)
                                                              : combine_rows(rows, w, p.position));
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"mx_quantize", (PyCFunction)(void (*)(void))mx_quantize, METH_FASTCALL, nullptr},
    {"mx_dequantize", (PyCFunction)(void (*)(void))mx_dequantize, METH_FASTCALL, nullptr},
    {"mx_linear", (PyCFunction)(void (*)(void))mx_linear, METH_FASTCALL, nullptr},
    {"mx_expert_linear", (PyCFunction)(void (*)(void))mx_expert_linear, METH_FASTCALL, nullptr},
    {"expert_sort", (PyCFunction)(void (*)(void))expert_sort, METH_FASTCALL, nullptr},
    {"expert_gather", (PyCFunction)(void (*)(void))expert_gather, METH_FASTCALL, nullptr},
    {"expert_combine", (PyCFunction)(void (*)(void))expert_combine, METH_FASTCALL, nullptr},
    {"w4a4", (PyCFunction)(void (*)(void))w4a4, METH_FASTCALL, nullptr},
    {"w8a8", (PyCFunction)(void (*)(void))w8a8, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// ABI_VERSION: of the library's signatures this module was compiled with.
PyMODINIT_FUNC PyInit__host(void) {
    PyObject* m = PyModule_Create(&module);
    if (m != nullptr && PyModule_AddIntConstant(m, "ABI_VERSION", CR_ABI_VERSION) != 0) Py_CLEAR(m);
    return m;
}
