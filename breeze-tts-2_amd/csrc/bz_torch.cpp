// Torch binding of the calls whose host work can take longer than their
// kernels: products over tiled weights, and quantising rows.  In Python the
// checks, the descriptor, the output and the library call of a decode step's
// product take 7.6 us; here they take 5.1 us, 2.6 of them HIP's launch (quantise
// 8.0 -> 4.8, read back 6.7 -> 4.4, a product of quantised rows 7.9 -> 4.8).
//
// Every function takes its arguments as the Python function of its name does
// and returns None where one of them needs converting or copying, another
// device, a plan that is not there yet, or refusing: the Python function then
// does that, or raises.  So nothing here reports an error but those of torch (no
// memory) and of the workspace.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "bz_mx.h"

namespace {

// entries of the library, which Python has loaded
decltype(&bz_gemv) f_gemv;
decltype(&bz_mx_gemv) f_mx_gemv;
decltype(&bz_mx_gemm) f_mx_gemm;
decltype(&bz_gemm_tiled) f_gemm;
decltype(&bz_gemm_workspace) f_gemm_workspace;
decltype(&bz_tiled_bytes) f_tiled_bytes;
decltype(&bz_mx_quantize) f_quantize;
decltype(&bz_mx_dequantize) f_dequantize;
PyObject* tiled_key;  // "tiled"

// A tensor (no subclass, whose operations may mean something else) on the
// current device, or null.
const at::Tensor* gpu(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.get_device() == c10::hip::current_device() ? &t : nullptr;
}

bool aligned(const at::Tensor& t, uintptr_t to) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % to == 0; }

// bz_dtype of bf16 and fp32, else -1.
int dtype_of(at::ScalarType t) { return t == at::kBFloat16 ? BZ_DT_BF16 : t == at::kFloat ? BZ_DT_F32 : -1; }
int dtype_of(PyObject* o) { return THPDtype_Check(o) ? dtype_of(reinterpret_cast<THPDtype*>(o)->scalar_type) : -1; }

// x type of bz_mx_quantize, else -1.
int x_dtype(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? BZ_MX_F16 : dtype_of(t.scalar_type()); }

int elem(PyObject* o) {
    if (!PyUnicode_Check(o)) return -1;
    if (PyUnicode_CompareWithASCIIString(o, "e2m1") == 0) return BZ_MX_E2M1;
    return PyUnicode_CompareWithASCIIString(o, "e4m3") == 0 ? BZ_MX_E4M3 : -1;
}

// Whether autograd follows t, backward or forward.
bool followed(const at::Tensor& t) {
    return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined();
}

// A non-negative int, else -1.
int64_t number(PyObject* o) {
    if (!PyLong_Check(o)) return -1;
    int overflow = 0;
    return PyLong_AsLongLongAndOverflow(o, &overflow);
}

void* stream() { return c10::hip::getCurrentHIPStream().stream(); }

// Allocation and launch can wait for the GPU, and what it waits for may need
// the interpreter (a host function of a stream).
struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};

// Address and bytes of `need` bytes of workspace from f(device index, stream,
// need), which Python keeps; false with an error set.
bool workspace(PyObject* f, const at::Tensor& x, int64_t need, void*& at, size_t& bytes) {
    PyObject* r = PyObject_CallFunction(f, "iKL", (int)x.get_device(), (unsigned long long)stream(), (long long)need);
    unsigned long long p = 0, n = 0;
    const bool ok = r && PyArg_ParseTuple(r, "KK", &p, &n);
    Py_XDECREF(r);
    at = reinterpret_cast<void*>(p);
    bytes = (size_t)n;
    return ok;
}

bool is_tiled(int64_t wfmt) {
    return (wfmt >= BZ_W_INT4_TILED && wfmt <= BZ_W_FP8_TILED_PAIRED) || wfmt == BZ_W_MXFP4_TILED ||
           wfmt == BZ_W_MXFP4_TILED_PAIRED;
}

// The plan of a product that gemv._plan_tiled has put into the launch-shape
// table of the device: (output columns, bytes of the weight, launch shape,
// workspace bytes).  Borrowed; null without an error where there is none.
PyObject* plan_of(PyObject* tables, PyObject* archs, int64_t index, int64_t wfmt, int64_t n, int64_t k, int64_t epi,
                  bool norm, int64_t m) {
    PyObject* at = PyLong_FromLongLong(index);
    PyObject* arch = at ? PyDict_GetItemWithError(archs, at) : nullptr;
    Py_XDECREF(at);
    PyObject* table = arch ? PyDict_GetItemWithError(tables, arch) : nullptr;
    if (!table || !PyDict_Check(table)) return nullptr;
    PyObject* key = Py_BuildValue("(OLLLLiL)", tiled_key, (long long)wfmt, (long long)n, (long long)k, (long long)epi,
                                  (int)norm, (long long)m);
    PyObject* plan = key ? PyDict_GetItemWithError(table, key) : nullptr;
    Py_XDECREF(key);
    return plan && PyTuple_Check(plan) && PyTuple_GET_SIZE(plan) == 4 ? plan : nullptr;
}

// gemv(tables, archs, workspace, x, w, wfmt, n, gamma, eps, epilogue, residual, out_dtype)
PyObject* gemv(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 12) Py_RETURN_NONE;
    const at::Tensor *x = gpu(a[3]), *w = gpu(a[4]);
    const int64_t wfmt = number(a[5]), n = number(a[6]), epi = number(a[9]);
    const int odt = dtype_of(a[11]);
    const bool norm = a[7] != Py_None;
    if (!x || !w || x->dim() != 2 || x->scalar_type() != at::kBFloat16 || odt < 0 || n < 1 || !is_tiled(wfmt) ||
        epi < 0 || !PyFloat_Check(a[8]) || !PyDict_Check(a[0]) || !PyDict_Check(a[1]))
        Py_RETURN_NONE;
    const int64_t M = x->size(0), K = x->size(1), ld = x->stride(0);
    if (M < 1 || M > 32 || K < 1 || x->stride(1) != 1 || ld < K || ld % 8 || !aligned(*x, 16)) Py_RETURN_NONE;
    PyObject* plan = plan_of(a[0], a[1], x->get_device(), wfmt, n, K, epi, norm, M);
    if (!plan) {
        if (PyErr_Occurred()) return nullptr;
        Py_RETURN_NONE;
    }
    const int64_t n_out = number(PyTuple_GET_ITEM(plan, 0)), need = number(PyTuple_GET_ITEM(plan, 3));
    PyObject* cfg = PyTuple_GET_ITEM(plan, 2);
    if (!w->is_contiguous() || (int64_t)w->nbytes() != number(PyTuple_GET_ITEM(plan, 1)) ||
        need < 0 || !PyTuple_Check(cfg) || PyTuple_GET_SIZE(cfg) != 5)
        Py_RETURN_NONE;
    bz_gemv_desc d{};
    if (norm) {
        const at::Tensor* g = gpu(a[7]);
        if (!g || g->scalar_type() != at::kBFloat16 || g->numel() != K || !g->is_contiguous()) Py_RETURN_NONE;
        d.gamma = g->data_ptr();
    }
    if (epi == BZ_EPI_RESIDUAL) {
        const at::Tensor* r = a[10] == Py_None ? nullptr : gpu(a[10]);
        if (!r || r->dim() != 2 || r->size(0) != M || r->size(1) != n_out || r->stride(1) != 1) Py_RETURN_NONE;
        d.residual_dtype = dtype_of(r->scalar_type());
        if (d.residual_dtype < 0) Py_RETURN_NONE;
        d.residual = r->data_ptr();
        d.ldr = r->stride(0);
    }
    d.abi_version = BZ_ABI_VERSION;
    d.M = (int32_t)M;
    d.N = (int32_t)n;
    d.K = (int32_t)K;
    d.group = 128;
    d.wfmt = (int32_t)wfmt;
    d.epilogue = (int32_t)epi;
    d.out_dtype = odt;
    d.cfg_depth = (int32_t)number(PyTuple_GET_ITEM(cfg, 0));
    d.cfg_waves = (int32_t)number(PyTuple_GET_ITEM(cfg, 1));
    d.cfg_tiles = (int32_t)number(PyTuple_GET_ITEM(cfg, 2));
    d.cfg_path = (int32_t)number(PyTuple_GET_ITEM(cfg, 3));
    d.cfg_slices = (int32_t)number(PyTuple_GET_ITEM(cfg, 4));
    d.eps = (float)PyFloat_AS_DOUBLE(a[8]);
    d.x = x->data_ptr();
    d.ldx = ld;
    d.w = w->data_ptr();
    d.ldo = n_out;
    // (last: it runs Python, where another thread may replace the table that
    // plan and cfg are borrowed from)
    if (need && !workspace(a[2], *x, need, d.workspace, d.workspace_bytes)) return nullptr;
    at::Tensor out;
    int rc;
    {
        NoGil no_gil;
        out = at::empty({M, n_out}, x->options().dtype(odt == BZ_DT_F32 ? at::kFloat : at::kBFloat16));
        d.out = out.data_ptr();
        rc = f_gemv(&d, stream());
    }
    if (rc != BZ_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// quantize_mx(x, elem)
PyObject* quantize_mx(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    const at::Tensor* x = count == 2 ? gpu(a[0]) : nullptr;
    const int el = x ? elem(a[1]) : -1;
    if (el < 0 || x->dim() != 2 || followed(*x)) Py_RETURN_NONE;
    const int dt = x_dtype(*x);
    const int64_t M = x->size(0), K = x->size(1), ld = M == 1 ? K : x->stride(0);
    if (dt < 0 || M < 1 || K < 1 || K % 32 || M > INT32_MAX || K > INT32_MAX || x->stride(1) != 1 || ld < K)
        Py_RETURN_NONE;
    at::Tensor codes, scales;
    int rc;
    {
        NoGil no_gil;
        codes = el == BZ_MX_E2M1 ? at::empty({M, K / 2}, x->options().dtype(at::kByte))
                                 : at::empty({M, K}, x->options().dtype(at::kFloat8_e4m3fn));
        scales = at::empty({M, K / 32}, x->options().dtype(at::kByte));
        rc = f_quantize(x->data_ptr(), dt, ld, (int32_t)M, (int32_t)K, el, BZ_MX_ROWS, codes.data_ptr(),
                        scales.data_ptr(), stream());
    }
    if (rc != BZ_OK) Py_RETURN_NONE;
    PyObject* r = PyTuple_New(2);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(codes)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(scales)));
    return r;
    END_HANDLE_TH_ERRORS
}

// dequantize_mx(codes, scales, elem, dtype)
PyObject* dequantize_mx(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 4) Py_RETURN_NONE;
    const at::Tensor *codes = gpu(a[0]), *scales = gpu(a[1]);
    const int el = elem(a[2]), dt = dtype_of(a[3]);
    if (!codes || !scales || el < 0 || dt < 0 || codes->dim() != 2 || scales->dim() != 2) Py_RETURN_NONE;
    const bool e4m3 = el == BZ_MX_E4M3;
    if (!(codes->scalar_type() == at::kByte || (e4m3 && codes->scalar_type() == at::kFloat8_e4m3fn)) ||
        scales->scalar_type() != at::kByte || !codes->is_contiguous() || !scales->is_contiguous() || !aligned(*codes, 4))
        Py_RETURN_NONE;
    const int64_t M = codes->size(0), K = codes->size(1) * (e4m3 ? 1 : 2);
    if (M < 1 || K < 1 || K % 32 || M > INT32_MAX || K > INT32_MAX || scales->size(0) != M || scales->size(1) != K / 32)
        Py_RETURN_NONE;
    at::Tensor out;
    int rc;
    {
        NoGil no_gil;
        out = at::empty({M, K}, codes->options().dtype(dt == BZ_DT_F32 ? at::kFloat : at::kBFloat16));
        rc = f_dequantize(codes->data_ptr(), scales->data_ptr(), el, (int32_t)M, (int32_t)K, out.data_ptr(), dt, K,
                          stream());
    }
    if (rc != BZ_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// mx_linear(plans, workspace, x, w, n, elem, residual, out_dtype).  plans:
// (elem, M, n, K) -> (bytes of the weight, whether one launch takes bf16 rows as
// they are, workspace bytes, bytes of the quantised rows).
PyObject* mx_linear(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 8 || !PyDict_Check(a[0])) Py_RETURN_NONE;
    const at::Tensor *x = gpu(a[2]), *w = gpu(a[3]);
    const int64_t n = number(a[4]);
    const int el = elem(a[5]), odt = dtype_of(a[7]);
    if (!x || !w || n < 1 || el < 0 || odt < 0 || x->dim() != 2 || followed(*x))
        Py_RETURN_NONE;
    const int dt = x_dtype(*x);
    const int64_t M = x->size(0), K = x->size(1), ld = M == 1 ? K : x->stride(0);
    if (dt < 0 || M < 1 || M > INT32_MAX || x->stride(1) != 1 || ld < K) Py_RETURN_NONE;
    PyObject* key = Py_BuildValue("(iLLL)", el, (long long)M, (long long)n, (long long)K);
    PyObject* plan = key ? PyDict_GetItemWithError(a[0], key) : nullptr;
    Py_XDECREF(key);
    if (!plan || !PyTuple_Check(plan) || PyTuple_GET_SIZE(plan) != 4) {
        if (PyErr_Occurred()) return nullptr;
        Py_RETURN_NONE;
    }
    const bool few = PyTuple_GET_ITEM(plan, 1) == Py_True;
    const int64_t need = number(PyTuple_GET_ITEM(plan, 2)), rows = number(PyTuple_GET_ITEM(plan, 3));
    if (!w->is_contiguous() || (int64_t)w->nbytes() != number(PyTuple_GET_ITEM(plan, 0)) || need < 0 || rows < 0 ||
        (few && (dt != BZ_DT_BF16 || ld % 8 || M * ld >= 1 << 30 || !aligned(*x, 16))))
        Py_RETURN_NONE;
    const at::Tensor* r = a[6] == Py_None ? nullptr : gpu(a[6]);
    int rdt = 0;
    if (a[6] != Py_None) {
        rdt = r ? dtype_of(r->scalar_type()) : -1;
        if (rdt < 0 || r->dim() != 2 || r->size(0) != M || r->size(1) != n || r->stride(1) != 1 ||
            (M > 1 && r->stride(0) < n) || followed(*r))
            Py_RETURN_NONE;
    }
    const void* res = r ? r->data_ptr() : nullptr;
    const int64_t ldr = r && M > 1 ? r->stride(0) : n;
    void* ws = nullptr;
    size_t bytes = 0;
    if (need && !workspace(a[1], *x, need, ws, bytes)) return nullptr;
    at::Tensor out;
    int rc;
    {
        NoGil no_gil;
        out = at::empty({M, n}, x->options().dtype(odt == BZ_DT_F32 ? at::kFloat : at::kBFloat16));
        if (few) {
            rc = f_mx_gemv(el, x->data_ptr(), ld, (int32_t)M, w->data_ptr(), (int32_t)n, (int32_t)K, res, rdt, ldr,
                           out.data_ptr(), odt, n, ws, bytes, 0, stream());
        } else {
            at::Tensor q = at::empty({rows}, x->options().dtype(at::kByte));
            rc = f_quantize(x->data_ptr(), dt, ld, (int32_t)M, (int32_t)K, el, BZ_MX_TILED, q.data_ptr(), nullptr,
                            stream());
            if (rc == BZ_OK)
                rc = f_mx_gemm(el, q.data_ptr(), (int32_t)M, w->data_ptr(), (int32_t)n, (int32_t)K, res, rdt, ldr,
                               out.data_ptr(), odt, n, ws, bytes, 0, stream());
        }
    }
    if (rc != BZ_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// dequant_matmul(x, w, wfmt, n, k) of an x without forward gradients
PyObject* dequant_matmul(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 5) Py_RETURN_NONE;
    const at::Tensor *x = gpu(a[0]), *w = gpu(a[1]);
    const int64_t wfmt = number(a[2]), n = number(a[3]), k = number(a[4]);
    if (!x || !w || (wfmt != BZ_W_INT4_TILED && wfmt != BZ_W_FP8_TILED && wfmt != BZ_W_MXFP4_TILED) || n < 1 ||
        n > INT32_MAX || k < 1 || k > INT32_MAX || x->dim() != 2 || x->size(1) != k ||
        x->scalar_type() != at::kBFloat16 || (x->requires_grad() && c10::GradMode::is_enabled()))
        Py_RETURN_NONE;
    const int64_t M = x->size(0), ld = x->stride(0);
    const size_t bytes = f_tiled_bytes((int32_t)wfmt, (int32_t)n, (int32_t)k);
    if (M < 1 || M > INT32_MAX || x->stride(1) != 1 || ld < k || ld > 1 << 22 || ld % 8 || !aligned(*x, 16) || !bytes ||
        !w->is_contiguous() || w->nbytes() != bytes)
        Py_RETURN_NONE;
    at::Tensor out;
    int rc;
    {
        NoGil no_gil;
        out = at::empty({M, n}, x->options());
        const size_t need = f_gemm_workspace((int32_t)wfmt, (int32_t)M, (int32_t)n, (int32_t)k, 0);
        // from the caching allocator: its memory is reused in stream order
        at::Tensor sums;
        if (need) sums = at::empty({(int64_t)need}, x->options().dtype(at::kByte));
        rc = f_gemm((int32_t)wfmt, x->data_ptr(), ld, (int32_t)M, w->data_ptr(), (int32_t)n, (int32_t)k, out.data_ptr(), n,
                    BZ_DT_BF16, need ? sums.data_ptr() : nullptr, need, 0, stream());
    }
    if (rc != BZ_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// bind(addresses): of the library's entries, in this order
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long p[8];
    if (!PyArg_ParseTuple(args, "KKKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7)) return nullptr;
    f_gemv = reinterpret_cast<decltype(f_gemv)>(p[0]);
    f_mx_gemv = reinterpret_cast<decltype(f_mx_gemv)>(p[1]);
    f_mx_gemm = reinterpret_cast<decltype(f_mx_gemm)>(p[2]);
    f_quantize = reinterpret_cast<decltype(f_quantize)>(p[3]);
    f_dequantize = reinterpret_cast<decltype(f_dequantize)>(p[4]);
    f_gemm = reinterpret_cast<decltype(f_gemm)>(p[5]);
    f_gemm_workspace = reinterpret_cast<decltype(f_gemm_workspace)>(p[6]);
    f_tiled_bytes = reinterpret_cast<decltype(f_tiled_bytes)>(p[7]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"gemv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gemv)), METH_FASTCALL, nullptr},
    {"mx_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mx_linear)), METH_FASTCALL, nullptr},
    {"dequant_matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequant_matmul)), METH_FASTCALL, nullptr},
    {"quantize_mx", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(quantize_mx)), METH_FASTCALL, nullptr},
    {"dequantize_mx", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequantize_mx)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bztorch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bztorch() {
    tiled_key = PyUnicode_InternFromString("tiled");
    return tiled_key ? PyModule_Create(&module) : nullptr;
}
