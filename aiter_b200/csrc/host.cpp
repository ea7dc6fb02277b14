// CPython extension _aiter_b200_host: the host side of the operators with a fused epilogue, the norms and the gated activation.  A call
// allocates what it returns, fills the descriptors and enters the library (include/aiter_b200.h) without going back to Python: for one
// token the kernels take 2 to 10 us, and the same steps in Python took 7 to 12 (norm of one row of 4096: 12.3, of them 3.8 in the
// library).  Checks of what the arguments mean stay in Python and in the library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/aiter_b200.h"

#include <limits>
#include <type_traits>

namespace {

using Desc = aiter_tensor_t;
// the library's functions, with the types that the public header declares
#define ENTRY(name) decltype(&name)

struct Bound
{
    ENTRY(aiter_b200_gated_residual_norm) norm;
    ENTRY(aiter_b200_act_and_mul) act;
    ENTRY(aiter_b200_gemm_a16w16_fused) gemm16;
    ENTRY(aiter_b200_gemm_a8w8_mxfp8_fused) gemm8;
    ENTRY(aiter_b200_gemm_a4w4_fused) gemm4;
    ENTRY(aiter_b200_gemm_a4w4_fused_workspace) workspace;
    int dtypes[64]; // library's id of an ATen scalar type, -1: none
    at::ScalarType fp4x2, fp8, e8m0; // of MX operands and their scales
} bound = {};
PyObject* unsupported = nullptr; // raises, naming the type

// A tensor argument (None: absent) and its descriptor
struct Arg
{
    Desc d;
    Desc* ptr = nullptr;

    void set(const at::Tensor& t)
    {
        const auto type = static_cast<int>(t.scalar_type());
        const int id    = type >= 0 && type < 64 ? bound.dtypes[type] : -1;
        if(id < 0)
        {
            PyObject* r = PyObject_CallOneArg(unsupported, reinterpret_cast<PyObject*>(torch::getTHPDtype(t.scalar_type())));
            Py_XDECREF(r);
            if(r != nullptr)
                PyErr_SetString(PyExc_TypeError, "unsupported tensor type");
            throw python_error();
        }
        const int64_t n = t.dim();
        TORCH_CHECK(n <= 8, "aiter_tensor_t supports at most 8 dims, got ", n);
        d.ptr    = const_cast<void*>(t.const_data_ptr());
        d.numel_ = static_cast<size_t>(t.numel());
        d.ndim   = static_cast<int>(n);
        const auto sizes = t.sizes(), strides = t.strides();
        for(int64_t i = 0; i < n; ++i)
            d.shape[i] = sizes[i], d.strides[i] = strides[i];
        for(int64_t i = n; i < 8; ++i)
            d.shape[i] = d.strides[i] = 0;
        d.dtype_    = static_cast<AiterDtype>(id);
        d.device_id = t.is_cuda() ? static_cast<int>(t.get_device()) : -1;
        ptr         = &d;
    }
    explicit Arg(const at::Tensor& t)
    {
        if(t.defined())
            set(t);
    }
    explicit Arg(PyObject* o)
    {
        if(o == Py_None)
            return;
        TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a Tensor or None, got ", Py_TYPE(o)->tp_name);
        set(THPVariable_Unpack(o));
    }
    Arg(const Arg&) = delete;
};

const at::Tensor& tensor(PyObject* o)
{
    TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a Tensor, got ", Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
at::Tensor rows_like(const at::Tensor& t, int64_t m, int64_t n, PyObject* dtype)
{
    auto options = t.options();
    if(dtype != Py_None)
    {
        TORCH_CHECK_TYPE(THPDtype_Check(dtype), "expected a torch.dtype");
        options = options.dtype(reinterpret_cast<THPDtype*>(dtype)->scalar_type);
    }
    return at::empty({m, n}, options);
}
// Data and scale tensors of an MX output [m, n], shaped as per_1x32_mx_quant_hip shapes them for the layout
void mx_out(const at::Tensor& x, int64_t m, int64_t n, long bits, long layout, at::Tensor& y, at::Tensor& scale)
{
    int64_t rows = m, blocks = n / 32;
    if(layout == 1)
        rows = (m + 255) / 256 * 256, blocks = (blocks + 7) / 8 * 8;
    else if(layout == 2)
        rows = (m + 31) / 32 * 32;
    y     = at::empty({m, bits == 4 ? n / 2 : n}, x.options().dtype(bits == 4 ? bound.fp4x2 : bound.fp8));
    scale = at::empty({rows, blocks}, x.options().dtype(bound.e8m0));
}
PyObject* wrap(at::Tensor& t) { return t.defined() ? THPVariable_Wrap(std::move(t)) : Py_NewRef(Py_None); }
long integer(PyObject* o)
{
    const long v = PyLong_AsLong(o);
    if(v == -1 && PyErr_Occurred())
        throw python_error();
    return v;
}
float number(PyObject* o)
{
    const double v = PyFloat_AsDouble(o);
    if(v == -1.0 && PyErr_Occurred())
        throw python_error();
    return static_cast<float>(v);
}
void* address(PyObject* o)
{
    if(o == Py_None)
        return nullptr;
    void* p = PyLong_AsVoidPtr(o);
    if(p == nullptr && PyErr_Occurred())
        throw python_error();
    return p;
}
void count(Py_ssize_t got, Py_ssize_t want) { TORCH_CHECK_TYPE(got == want, "expected ", want, " arguments, got ", got); }

// Every function below returns its tensors, or None when the library refused the call (its message is read by the caller).

// norm(x, residual, weight, bias, gate, post_weight, post_bias, residual_out, bits, otype, residual_scale, weight_offset, eps, layer,
//      post, layout, stream) -> (y, scale, h); bits: 0, or 4 or 8 for an MX output; scale is None without it, h where it would be a copy of x
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    count(n, 17);
    const at::Tensor& x = tensor(a[0]);
    TORCH_CHECK(x.dim() == 2, "gated_residual_norm: x must have two dimensions");
    const long bits = integer(a[8]), layout = integer(a[15]);
    const bool post = integer(a[14]) != 0;
    at::Tensor h, y, sf;
    if(a[7] != Py_None)
        h = tensor(a[7]);
    else if(a[1] != Py_None || a[4] != Py_None || post)
        h = rows_like(a[1] != Py_None ? tensor(a[1]) : x, x.size(0), x.size(1), Py_None);
    if(bits != 0)
        mx_out(x, x.size(0), x.size(1), bits, layout, y, sf);
    else
        y = rows_like(x, x.size(0), x.size(1), a[9]);
    Arg dx(x), dr(a[1]), dw(a[2]), db(a[3]), dg(a[4]), dpw(a[5]), dpb(a[6]), dy(y), ds(sf), dh(h);
    const float scale = number(a[10]), offset = number(a[11]), eps = number(a[12]);
    const int layer    = static_cast<int>(integer(a[13]));
    void* const stream = address(a[16]);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = bound.norm(dy.ptr, ds.ptr, dh.ptr, dx.ptr, dr.ptr, dw.ptr, db.ptr, dg.ptr, dpw.ptr, dpb.ptr, scale, offset, eps, layer, post, static_cast<int>(layout), stream);
    Py_END_ALLOW_THREADS
    if(rc != 0)
        Py_RETURN_NONE;
    return Py_BuildValue("NNN", wrap(y), wrap(sf), wrap(h));
    END_HANDLE_TH_ERRORS
}

// act(x, y, bits, otype, activation, layout, stream) -> (y, scale); y is given for the out-forms
PyObject* act(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    count(n, 7);
    const at::Tensor& x = tensor(a[0]);
    TORCH_CHECK(x.dim() == 2, "act_and_mul: x must have two dimensions");
    const long bits = integer(a[2]), layout = integer(a[5]);
    at::Tensor y, sf;
    if(bits != 0)
        mx_out(x, x.size(0), x.size(1) / 2, bits, layout, y, sf);
    else
        y = a[1] != Py_None ? tensor(a[1]) : rows_like(x, x.size(0), x.size(1) / 2, a[3]);
    Arg dx(x), dy(y), ds(sf);
    const int activation = static_cast<int>(integer(a[4]));
    void* const stream = address(a[6]);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = bound.act(dy.ptr, ds.ptr, dx.ptr, activation, static_cast<int>(layout), stream);
    Py_END_ALLOW_THREADS
    if(rc != 0)
        Py_RETURN_NONE;
    return Py_BuildValue("NN", wrap(y), wrap(sf));
    END_HANDLE_TH_ERRORS
}

// gemm(bits, A, B, A_scale, B_scale, bias, residual, out, otype, activation, flag, name, stream) -> out; bits of an element of A: 16, 8
// or 4; flag: bpreshuffle (16, 4) or a_preshuffle (8); name: bytes or None
PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    count(n, 13);
    const long bits     = integer(a[0]);
    const at::Tensor& A = tensor(a[1]);
    const at::Tensor& B = tensor(a[2]);
    TORCH_CHECK(A.dim() == 2 && B.dim() == 2, "gemm: A and B must have two dimensions");
    at::Tensor out = a[7] != Py_None ? tensor(a[7]) : rows_like(A, A.size(0), B.size(0), a[8]);
    at::Tensor workspace;
    Arg dA(A), dB(B), dsa(a[3]), dsb(a[4]), dbias(a[5]), dres(a[6]), dout(out), dws(Py_None);
    if(bits == 4 && A.size(0) >= 1024)
    {
        // tall problems re-lay the block scales once per call, in memory of this call's own (two captured graphs share none)
        // (sizes that no int holds are the library's to refuse)
        constexpr int64_t most = std::numeric_limits<int>::max();
        const bool fit         = A.size(0) <= most && B.size(0) <= most && B.size(1) <= most / 2;
        const long long bytes  = fit ? bound.workspace(static_cast<int>(A.size(0)), static_cast<int>(B.size(0)), static_cast<int>(2 * B.size(1))) : 0;
        if(bytes > 0)
        {
            workspace = at::empty({static_cast<int64_t>(bytes)}, A.options().dtype(at::kByte));
            dws.set(workspace);
        }
    }
    const int activation = static_cast<int>(integer(a[9])), flag = PyObject_IsTrue(a[10]);
    const char* name = nullptr;
    if(a[11] != Py_None && (name = PyBytes_AsString(a[11])) == nullptr)
        throw python_error();
    void* const stream = address(a[12]);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = bits == 16  ? bound.gemm16(dA.ptr, dB.ptr, dbias.ptr, dres.ptr, dout.ptr, activation, flag, name, stream)
         : bits == 8 ? bound.gemm8(dA.ptr, dB.ptr, dsa.ptr, dsb.ptr, dbias.ptr, dres.ptr, dout.ptr, activation, flag, name, stream)
                     : bound.gemm4(dA.ptr, dB.ptr, dsa.ptr, dsb.ptr, dbias.ptr, dres.ptr, dout.ptr, dws.ptr, activation, flag, name, stream);
    Py_END_ALLOW_THREADS
    if(rc != 0)
        Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// bind(norm, act, gemm16, gemm8, gemm4, workspace: addresses in the library, dtypes: {torch.dtype: id}, unsupported: callable, fp4x2, fp8,
//      e8m0: torch.dtype)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    count(n, 11);
    auto entry = [&](auto& function, int i) { function = reinterpret_cast<std::remove_reference_t<decltype(function)>>(address(a[i])); };
    entry(bound.norm, 0);
    entry(bound.act, 1);
    entry(bound.gemm16, 2);
    entry(bound.gemm8, 3);
    entry(bound.gemm4, 4);
    entry(bound.workspace, 5);
    for(int& id : bound.dtypes)
        id = -1;
    PyObject *key, *value;
    Py_ssize_t pos = 0;
    TORCH_CHECK_TYPE(PyDict_Check(a[6]), "dtypes must be a dict");
    while(PyDict_Next(a[6], &pos, &key, &value))
    {
        TORCH_CHECK_TYPE(THPDtype_Check(key), "dtypes must map torch.dtype");
        const int type = static_cast<int>(reinterpret_cast<THPDtype*>(key)->scalar_type);
        if(type >= 0 && type < 64)
            bound.dtypes[type] = static_cast<int>(integer(value));
    }
    Py_XSETREF(unsupported, Py_NewRef(a[7]));
    for(int i = 8; i < 11; ++i)
    {
        TORCH_CHECK_TYPE(THPDtype_Check(a[i]), "expected a torch.dtype");
        (i == 8 ? bound.fp4x2 : i == 9 ? bound.fp8 : bound.e8m0) = reinterpret_cast<THPDtype*>(a[i])->scalar_type;
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(norm), METHOD(act), METHOD(gemm), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_aiter_b200_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__aiter_b200_host() { return PyModule_Create(&module); }
