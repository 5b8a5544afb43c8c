// nt_torch.cpp -- the usual calls of the texel-layer operators from torch tensors, without the host
// time of the Python wrappers (neural_textures_b200/layers.py), of which this is a shortcut: a function
// here takes plain CUDA tensors of the current device and torch's current stream, allocates the results,
// fills the parameter block and calls the C ABI.  Whatever is not that, invalid arguments included, it leaves
// to the wrapper by returning None.  It computes nothing itself.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "nt_capi.h"

namespace {

// A plain strided CUDA tensor on `device`, or null.
const at::Tensor *cuda_tensor(PyObject *o, c10::DeviceIndex device)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided && t.get_device() == device ? &t : nullptr;
}

// The device of a CUDA tensor when it is the current one, else -1.
c10::DeviceIndex current_device_of(PyObject *o)
{
    if (!THPVariable_CheckExact(o) || !THPVariable_Unpack(o).is_cuda()) return -1;
    const c10::DeviceIndex device = c10::cuda::current_device();
    return THPVariable_Unpack(o).get_device() == device ? device : -1;
}

int layer_dtype(at::ScalarType t)
{
    return t == at::kHalf ? NT_DTYPE_F16 : t == at::kBFloat16 ? NT_DTYPE_BF16 : t == at::kFloat ? NT_DTYPE_F32 : -1;
}

// An optional fp32 vector of n elements.
bool vector_arg(PyObject *o, int64_t n, c10::DeviceIndex device, float *&out)
{
    out = nullptr;
    if (o == Py_None) return true;
    const at::Tensor *t = cuda_tensor(o, device);
    if (!t || t->scalar_type() != at::kFloat || t->numel() != n || !t->is_contiguous()) return false;
    out = static_cast<float *>(t->data_ptr());
    return true;
}

// A channels-last map with x's sizes and type.
bool map_arg(const at::Tensor &t, const at::Tensor &like, NtFeatureMap &out)
{
    const int64_t dims = t.dim();
    if (t.scalar_type() != like.scalar_type() || t.sizes() != like.sizes()) return false;
    if (t.stride(dims - 1) != 1 && t.size(dims - 1) > 1) return false;
    out = {t.data_ptr(), dims == 4 ? t.stride(0) : 0, t.stride(dims - 3), t.stride(dims - 2)};
    return true;
}

bool int_arg(PyObject *o, long low, long high, int32_t &out)
{
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    out = (int32_t)v;
    return v >= low && v <= high;
}

at::Tensor make(at::IntArrayRef size, at::ScalarType type, c10::DeviceIndex device)
{
    return at::Tensor(at::detail::empty_cuda(size, type, at::Device(at::kCUDA, device), std::nullopt));
}

// Sizes of x into the parameter block.
bool norm_sizes(const at::Tensor &x, PyObject *groups, PyObject *act, NtGroupNorm &p)
{
    const int64_t d = x.dim();
    if (d != 3 && d != 4) return false;
    for (int64_t i = 0; i < d; ++i)
        if (x.size(i) > 0x7fffffff) return false;
    p.images = d == 4 ? (int32_t)x.size(0) : 1;
    p.height = (int32_t)x.size(d - 3);
    p.width = (int32_t)x.size(d - 2);
    p.channels = (int32_t)x.size(d - 1);
    p.dtype = layer_dtype(x.scalar_type());
    return p.dtype >= 0 && int_arg(groups, 1, NT_GROUP_NORM_MAX_CHANNELS, p.groups) && int_arg(act, 0, 3, p.activation);
}

// The workspace of the call, kept in `ws` until its launch is queued.
bool norm_workspace(NtGroupNorm &p, bool backward, c10::DeviceIndex device, at::Tensor &ws)
{
    const size_t need = nt_group_norm_workspace_bytes(&p, backward);
    if (need) {
        ws = make({(int64_t)need}, at::kByte, device);
        p.workspace = ws.data_ptr();
        p.workspace_bytes = (int64_t)need;
    }
    return true;
}

template <class F>
nt_status without_gil(F f)
{
    PyThreadState *state = PyEval_SaveThread();
    const nt_status st = f();
    PyEval_RestoreThread(state);
    return st;
}

PyObject *tuple3(const at::Tensor &a, const at::Tensor &b, const at::Tensor &c)
{
    PyObject *t = PyTuple_New(3);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
    PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(c));
    return t;
}

// (x, groups, gamma, beta, activation, eps) -> (y, mean, rstd)
PyObject *group_norm(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 6) Py_RETURN_NONE;
    const c10::DeviceIndex device = current_device_of(a[0]);
    if (device < 0) Py_RETURN_NONE;
    const at::Tensor *x = cuda_tensor(a[0], device);
    NtGroupNorm p;
    std::memset(&p, 0, sizeof p);
    if (!x || !norm_sizes(*x, a[1], a[4], p) || !map_arg(*x, *x, p.x)) Py_RETURN_NONE;
    float *gamma, *beta;
    if (!vector_arg(a[2], p.channels, device, gamma) || !vector_arg(a[3], p.channels, device, beta) || !PyFloat_Check(a[5])) Py_RETURN_NONE;
    p.gamma = gamma;
    p.beta = beta;
    p.epsilon = (float)PyFloat_AS_DOUBLE(a[5]);
    at::Tensor ws, y = make(x->sizes(), x->scalar_type(), device);
    at::Tensor mean = make({p.images, p.groups}, at::kFloat, device), rstd = make({p.images, p.groups}, at::kFloat, device);
    map_arg(y, *x, p.y);
    p.mean = static_cast<float *>(mean.data_ptr());
    p.rstd = static_cast<float *>(rstd.data_ptr());
    norm_workspace(p, false, device, ws);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device);
    if (without_gil([&] { return nt_group_norm_forward(&p, stream); }) != NT_OK) Py_RETURN_NONE;
    return tuple3(y, mean, rstd);
    END_HANDLE_TH_ERRORS
}

// (dy, x, mean, rstd, groups, gamma, beta, activation) -> (dx, dgamma, dbeta)
PyObject *group_norm_backward(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 8) Py_RETURN_NONE;
    const c10::DeviceIndex device = current_device_of(a[1]);
    if (device < 0) Py_RETURN_NONE;
    const at::Tensor *dy = cuda_tensor(a[0], device), *x = cuda_tensor(a[1], device);
    NtGroupNorm p;
    std::memset(&p, 0, sizeof p);
    if (!x || !dy || !norm_sizes(*x, a[4], a[7], p) || !map_arg(*x, *x, p.x) || !map_arg(*dy, *x, p.dy)) Py_RETURN_NONE;
    float *gamma, *beta;
    const int64_t stats = (int64_t)p.images * p.groups;
    if (!vector_arg(a[2], stats, device, p.mean) || !vector_arg(a[3], stats, device, p.rstd) ||
        !vector_arg(a[5], p.channels, device, gamma) || !vector_arg(a[6], p.channels, device, beta))
        Py_RETURN_NONE;
    p.gamma = gamma;
    p.beta = beta;
    p.epsilon = 1.f;
    at::Tensor ws, dx = make(x->sizes(), x->scalar_type(), device);
    at::Tensor dgamma = make({p.channels}, at::kFloat, device), dbeta = make({p.channels}, at::kFloat, device);
    map_arg(dx, *x, p.dx);
    p.dgamma = static_cast<float *>(dgamma.data_ptr());
    p.dbeta = static_cast<float *>(dbeta.data_ptr());
    norm_workspace(p, true, device, ws);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device);
    if (without_gil([&] { return nt_group_norm_backward(&p, stream); }) != NT_OK) Py_RETURN_NONE;
    return tuple3(dx, dgamma, dbeta);
    END_HANDLE_TH_ERRORS
}

// A NtMx4Matrix packed as bytes (Mx4Tensor._packed), while it names the memory of its tensors, on `device`.
bool matrix_arg(PyObject *packed, PyObject *data, PyObject *scales, c10::DeviceIndex device, NtMx4Matrix &m)
{
    const at::Tensor *d = cuda_tensor(data, device), *s = cuda_tensor(scales, device);
    if (!d || !s || !PyBytes_Check(packed) || PyBytes_GET_SIZE(packed) != (Py_ssize_t)sizeof m) return false;
    std::memcpy(&m, PyBytes_AS_STRING(packed), sizeof m);
    return m.data == d->data_ptr() && m.scales == s->data_ptr();
}

// (codes, scales, rows, cols, block) -> packed NtMx4Matrix
PyObject *mx4_pack(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    NtMx4Matrix m;
    std::memset(&m, 0, sizeof m);
    if (n != 5 || !THPVariable_CheckExact(a[0]) || !THPVariable_CheckExact(a[1]) || !int_arg(a[2], 0, 0x7fffff00, m.rows) ||
        !int_arg(a[3], 1, 0x7fffff00, m.cols) || !int_arg(a[4], 16, 32, m.block) || m.block % 16)
        Py_RETURN_NONE;
    const at::Tensor &data = THPVariable_Unpack(a[0]), &scales = THPVariable_Unpack(a[1]);
    m.pitch = (int64_t)nt_mx4_pitch(m.cols);
    if (data.scalar_type() != at::kByte || data.dim() != 2 || data.size(0) < m.rows || data.size(1) < m.pitch ||
        (m.rows > 0 && data.stride(1) != 1) ||
        scales.scalar_type() != at::kByte || !scales.is_contiguous() || scales.device() != data.device() ||
        scales.numel() < (int64_t)nt_mx4_scales_bytes(m.rows, m.cols, m.block))
        Py_RETURN_NONE;
    if (m.rows > 1) m.pitch = data.stride(0);
    m.data = data.data_ptr();
    m.scales = scales.data_ptr();
    return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(&m), sizeof m);
    END_HANDLE_TH_ERRORS
}

// (x, block) -> (codes, scales, packed NtMx4Matrix)
PyObject *mx4_quantize(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 2) Py_RETURN_NONE;
    const c10::DeviceIndex device = current_device_of(a[0]);
    if (device < 0) Py_RETURN_NONE;
    const at::Tensor *x = cuda_tensor(a[0], device);
    NtMx4Matrix m;
    std::memset(&m, 0, sizeof m);
    if (!x || x->dim() != 2 || !int_arg(a[1], 16, 32, m.block) || m.block % 16 || x->size(0) > 0x7fffff00 || x->size(1) < 1 ||
        x->size(1) > 0x7fffff00 || layer_dtype(x->scalar_type()) < 0)
        Py_RETURN_NONE;
    m.rows = (int32_t)x->size(0);
    m.cols = (int32_t)x->size(1);
    m.pitch = (int64_t)nt_mx4_pitch(m.cols);
    at::Tensor data = make({m.rows, m.pitch}, at::kByte, device);
    at::Tensor scales = make({(int64_t)nt_mx4_scales_bytes(m.rows, m.cols, m.block)}, at::kByte, device);
    m.data = data.data_ptr();
    m.scales = scales.data_ptr();
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device);
    if (without_gil([&] {
            return nt_mx4_quantize(x->data_ptr(), layer_dtype(x->scalar_type()), x->stride(0), x->stride(1), &m, stream);
        }) != NT_OK)
        Py_RETURN_NONE;
    PyObject *t = PyTuple_New(3);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(data));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(scales));
    PyTuple_SET_ITEM(t, 2, PyBytes_FromStringAndSize(reinterpret_cast<const char *>(&m), sizeof m));
    return t;
    END_HANDLE_TH_ERRORS
}

at::ScalarType scalar_type(int32_t dtype) { return dtype == NT_DTYPE_F32 ? at::kFloat : dtype == NT_DTYPE_F16 ? at::kHalf : at::kBFloat16; }

// (packed, codes, scales, dtype) -> values
PyObject *mx4_dequantize(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 4) Py_RETURN_NONE;
    const c10::DeviceIndex device = current_device_of(a[1]);
    if (device < 0) Py_RETURN_NONE;
    NtMx4Matrix m;
    int32_t dtype;
    if (!matrix_arg(a[0], a[1], a[2], device, m) || !int_arg(a[3], 0, NT_DTYPE_BF16, dtype)) Py_RETURN_NONE;
    at::Tensor y = make({m.rows, m.cols}, scalar_type(dtype), device);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device);
    if (without_gil([&] { return nt_mx4_dequantize(&m, y.data_ptr(), dtype, m.cols, stream); }) != NT_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// (a packed, a codes, a scales, b packed, b codes, b scales, bias, activation, alpha, dtype) -> d
PyObject *mx4_product(PyObject *, PyObject *const *a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    if (n != 10) Py_RETURN_NONE;
    const c10::DeviceIndex device = current_device_of(a[1]);
    if (device < 0) Py_RETURN_NONE;
    NtMx4Matrix l, r;
    int32_t act, dtype;
    float *bias;
    if (!matrix_arg(a[0], a[1], a[2], device, l) || !matrix_arg(a[3], a[4], a[5], device, r) ||
        !vector_arg(a[6], r.rows, device, bias) || !int_arg(a[7], 0, 3, act) || !PyFloat_Check(a[8]) ||
        !int_arg(a[9], 0, NT_DTYPE_BF16, dtype))
        Py_RETURN_NONE;
    at::Tensor d = make({l.rows, r.rows}, scalar_type(dtype), device);
    const float alpha = (float)PyFloat_AS_DOUBLE(a[8]);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device);
    if (without_gil([&] { return nt_mx4_product(&l, &r, bias, act, alpha, d.data_ptr(), dtype, r.rows, stream); }) != NT_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(d);
    END_HANDLE_TH_ERRORS
}

using Fast = PyObject *(*)(PyObject *, PyObject *const *, Py_ssize_t);
PyMethodDef method(const char *name, Fast f)
{
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method("group_norm", group_norm),
                         method("group_norm_backward", group_norm_backward),
                         method("mx4_pack", mx4_pack),
                         method("mx4_quantize", mx4_quantize),
                         method("mx4_dequantize", mx4_dequantize),
                         method("mx4_product", mx4_product),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "nt_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit_nt_torch() { return PyModule_Create(&module); }
